"""A paged cache built on the CPU for tests, and plain 64-bit references of its three calls.

Every slot of the pool that no sequence holds is NaN (codes, scales and 16-bit
rows alike), so that a read of one shows.
"""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TOP = {torch.float16: 7, torch.bfloat16: 119}


def quantise(x):
    """e4m3 codes and e8m0 scales of rows, by exact 64-bit arithmetic on the CPU."""
    top, x = TOP[x.dtype], x.double()
    fine = torch.isfinite(x)
    amax = torch.where(fine, x, 0.0).abs().amax(-1)
    e = torch.full(amax.shape, -126.0, dtype=torch.float64)
    for k in range(-126, top):  # raised while a value passes 448 2^e
        e = torch.where(amax > 448 * 2.0 ** k, torch.tensor(k + 1.0, dtype=torch.float64), e)
    y = (x / torch.exp2(e)[..., None]).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.where(fine, torch.round(y / step) * step, math.nan)
    codes = y.float().to(torch.float8_e4m3fn)
    assert torch.equal(codes.double().nan_to_num(7.7), y.nan_to_num(7.7))
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


class Cache:
    """CPU tensors; rows(b) gives sequence b's K, V in 64 bits, [Hkv, len, D]."""

    def __init__(self, lens, hkv, d, page, dtype, q8, seed=0, news=None, width=None, gone=(), spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.d, self.page, self.dtype, self.q8 = lens, hkv, d, page, dtype, q8
        self.news = [1] * len(lens) if news is None else news
        need = [-(-n // page) for n in lens]
        self.width = max([1] + need) if width is None else width
        pool = sum(need) + 3
        order = torch.randperm(pool, generator=g).tolist()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.tensor([0] + self.news, dtype=torch.int32).cumsum(0).int()
        nan = torch.full((pool, hkv, page, d), math.nan, dtype=dtype)
        self.k, self.v, self.pages = nan.clone(), nan.clone(), pool
        self.rows = []  # per sequence [K, V] in the 16-bit type, [Hkv, len, D]
        for b, n in enumerate(lens):
            kv = [(torch.randn(hkv, n, d, generator=g) *
                   torch.exp(0.5 * spread * torch.randn(hkv, n, 1, generator=g))).to(dtype) for _ in "kv"]
            self.rows.append(kv)
            for i in range(min(need[b], self.width)):
                p = order.pop()
                self.table[b, i] = p
                part = slice(i * page, min(n, (i + 1) * page))
                for pool_t, x in ((self.k, kv[0]), (self.v, kv[1])):
                    pool_t[p, :, : part.stop - part.start] = x[:, part]
        self.ks = self.vs = None
        if q8:
            self.k, self.ks = quantise(self.k)
            self.v, self.vs = quantise(self.v)
            for s, c in ((self.ks, self.k), (self.vs, self.v)):
                s.view(torch.uint8)[torch.isnan(c.float()).all(-1)] = 255
            self.rows = [[x.double() if x.numel() == 0 else _through8(x) for x in kv] for kv in self.rows]
        else:
            self.rows = [[x.double() for x in kv] for kv in self.rows]
        for b, i in gone:
            self.table[b, i] = -1

    def held(self, b):
        """Which positions of sequence b are in a page, [len]."""
        pos = torch.arange(self.lens[b])
        ok = pos < self.width * self.page
        t = self.table[b][(pos // self.page).clamp(max=self.width - 1)]
        return ok & (t >= 0) & (t < self.pages)

    def args(self, device, strided=False):
        """(k, v, table, lens) and the keyword arguments of the calls, on `device`."""
        def put(x):
            if strided:  # [pages, page, Hkv, D] storage
                return x.transpose(1, 2).contiguous().to(device).transpose(1, 2)
            return x.to(device)
        kw = {}
        if self.q8:
            kw = {"k_scale": self.ks.to(device), "v_scale": self.vs.to(device)}
            if strided:
                kw = {n: t.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2)
                      .view(torch.float8_e8m0fnu) for n, t in kw.items()}
        return (put(self.k), put(self.v), self.table.to(device), self.seq_lens.to(device)), kw


def _through8(x):
    codes, scale = quantise(x)
    return codes.double() * scale.double()[..., None]


def attention(c, q, causal=True, scale=None):
    """O [T, Hq, D], LSE [Hq, T] in 64 bits, and the bounds of their errors.

    |O' - O| <= u (A + |O|) + f A + t, for A = sum_j p_j |v_j| (p the exact weights):
      u A     each weight rounded to the type (half a step u)
      u |O|   the result's rounding
      f A     32-bit sums over n keys and D products: a score is off by at most
              s = D 2^-24 scale sum |q k|, its weight by a factor e^(2s + 2^-22) (exp2 and the
              scaling round twice, in 32 bits, exponents up to 2^8: 2^-15), sums of n terms by
              n 2^-23 (numerator and denominator)
      t       float16: a weight below 2^-14 of the maximum is off by up to 2^-25 of it: 2^-25
              sum_j |v_j| / l, with l >= 1 in units of the largest weight
    and the LSE by 2s + n 2^-24 + 2^-15 + 2^-20 |LSE|.
    """
    t, hq, d = q.shape
    u = U[q.dtype]
    scale = 1 / math.sqrt(d) if scale is None else scale
    o = torch.zeros(t, hq, d, dtype=torch.float64)
    lse = torch.full((hq, t), -math.inf, dtype=torch.float64)
    o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    group = hq // c.hkv
    for b, n in enumerate(c.news):
        held = c.held(b)
        pos = torch.arange(c.lens[b])
        t0 = int(c.cu[b])
        k, v = c.rows[b]
        for h in range(hq):
            qb = q[t0:t0 + n, h].double()
            x = qb @ k[h // group].T * scale
            size = qb.abs() @ k[h // group].abs().T * abs(scale)
            row = torch.arange(n)[:, None] + c.lens[b] - n
            seen = held[None] & ((pos[None] <= row) if causal else torch.ones_like(row, dtype=torch.bool))
            x = x.masked_fill(~seen, -math.inf)
            if x.shape[1] == 0 or n == 0:
                continue
            m = x.amax(-1, keepdim=True)
            m = torch.where(m == -math.inf, 0.0, m)
            p = torch.exp(x - m)
            l = p.sum(-1, keepdim=True)
            some = l > 0
            w = torch.where(some, p / l, 0.0)
            vh = v[h // group]
            y = w @ vh
            s = (d * 2.0 ** -24 * size.masked_fill(~seen, 0.0).amax(-1, keepdim=True))
            keys = seen.sum(-1, keepdim=True)
            f = 2 * s + 2.0 ** -15 + keys * 2.0 ** -23
            a = w @ vh.abs()
            tiny = 0.0
            if q.dtype == torch.float16:
                tiny = torch.where(some, 2.0 ** -25 * (seen.double() @ vh.abs()) / l.clamp(min=1.0), 0.0)
            o[t0:t0 + n, h] = y
            o_tol[t0:t0 + n, h] = u * (a + y.abs()) + f * a * (1 + u) + tiny + 2.0 ** -25
            z = (m + torch.log(l))[:, 0]
            lse[h, t0:t0 + n] = z
            lse_tol[h, t0:t0 + n] = (2 * s + keys * 2.0 ** -24 + 2.0 ** -15)[:, 0] + 2.0 ** -20 * z.abs().nan_to_num(0.0, posinf=0.0)
    return o, lse, o_tol, lse_tol


def check(got, want, tol, what):
    got = got.double().cpu()
    err = (got - want).abs()
    bad = ~(err <= tol) & ~((got == want))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}, tolerance {tol.expand_as(want)[bad][0].item()}")
