"""Timing cases of the paged key/value cache: writing new tokens to it, reading it back, and the
attention of new tokens (a chunk of a prompt, or one generated token) over it.

A cache is a pool of pages, [pages, heads_kv, page_size, head_dim] for K and the same for V, in the
model's 16-bit type or in 8 bits (e4m3 codes, and a power-of-two scale for each token and head, e8m0).
`block_table[b]` lists the pages of sequence b in order, a negative entry being a page that is gone;
`seq_lens[b]` counts its tokens, the new ones included, which are its last ones;
`cu_seqlens[b] .. cu_seqlens[b + 1]` are their rows in Q, K and V ([tokens, heads, head_dim]).

  write   paged_cache_write: the new tokens' K and V into their pages
  read    paged_cache_read: every sequence's K and V out of its pages, [batch, heads_kv, longest, head_dim]
  attend  flash_attention_paged: softmax(scale Q K^T) V of the new tokens over their sequence's cache,
          token i of n seeing keys 0 .. seq_len - n + i, and the rows' log-sum-exp where a caller merges
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# The largest scale of a written row: 448 times it is finite in the rows' type.
TOP = {"fp16": 7, "bf16": 119}


def _fa():
    """The package, imported once, where its calls are the ones that run."""
    if not hasattr(_fa, "package"):
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "flash-attention-sm75-register-fused_amd", "src"))
        import flash_attention_sm75

        _fa.package = flash_attention_sm75
    return _fa.package


def _case(name, op, dtype, q8, b, hq, hkv, d, page, lo, hi, n, new="all", gone=False, lse=False):
    """`b` sequences of `lo` to `hi` tokens; `n` new tokens in each of them, or (new="one") in the
    first and one in the others; gone: the pages of the first tokens of every other sequence are."""
    c = {"op": op, "dtype": dtype, "q8": q8, "b": b, "hq": hq, "hkv": hkv, "d": d, "page": page,
         "lo": lo, "hi": hi, "n": n, "new": new, "gone": gone, "lse": lse}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one generated token of one sequence goes to its page: every layer and token, latency counts
        _case("write_token", "write", "bf16", False, 1, 14, 2, 64, 16, 4097, 4097, 1),
        # one token of each sequence of a serving batch, quantised on the way
        _case("write_batch_q8", "write", "fp16", True, 64, 32, 8, 128, 32, 512, 1024, 1),
        # the chunks of four prompts, quantised on the way
        _case("write_prompt_q8", "write", "bf16", True, 4, 32, 8, 128, 64, 2048, 4096, 2000),
        # a ragged batch's cache back as one padded tensor, from 8 bits (to move or to inspect it)
        _case("read_ragged_q8", "read", "bf16", True, 7, 14, 2, 64, 16, 1000, 8191, 1),
        # the same of a 16-bit cache of large heads
        _case("read_batch", "read", "fp16", False, 4, 32, 8, 128, 64, 4096, 8192, 1),
        # one generated token of one sequence: once per layer and token, latency counts
        _case("decode_token", "attend", "bf16", False, 1, 14, 2, 64, 16, 4097, 4097, 1),
        # one token of each sequence of a serving batch: streaming the cache
        _case("decode_batch", "attend", "fp16", False, 32, 32, 8, 128, 64, 4096, 8192, 1),
        # the same over 8 bits, half the bytes
        _case("decode_batch_q8", "attend", "bf16", True, 32, 32, 8, 128, 32, 4096, 8192, 1),
        # a few drafted tokens checked against a very long context in 8 bits
        _case("draft_long_q8", "attend", "bf16", True, 1, 32, 8, 128, 128, 131072, 131072, 4),
        # a later chunk of a long prompt, its log-sum-exp kept for a merge: the largest product
        _case("chunk_8192", "attend", "bf16", False, 1, 32, 8, 128, 64, 8192, 8192, 2048, lse=True),
        # odd chunks of three prompts of a small model over 8 bits, early pages gone
        _case("chunk_ragged_q8", "attend", "fp16", True, 3, 14, 2, 64, 16, 1777, 4000, 777, gone=True),
        # a serving step: one prompt's chunk among single tokens
        _case("mixed_step", "attend", "bf16", False, 16, 32, 8, 128, 16, 1000, 4096, 512, new="one"),
    ]


# (query heads, KV heads, head_dim) of the repository's configurations, tests and benchmark
HEADS = [(1, 1, 64), (8, 8, 64), (8, 8, 128), (12, 12, 64), (14, 2, 64), (16, 4, 128), (32, 8, 64),
         (32, 8, 128), (64, 8, 128)]


def _length(rng, lo, hi):
    """Spread over the logarithm; one in four a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(64, n // 64 * 64) if hi >= 64 and rng.random() < 1 / 4 else n


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
    hq, hkv, d = rng.choice(HEADS)
    dtype, q8 = rng.choice(["fp16", "bf16"]), rng.random() < 0.5
    page = rng.choice([16, 16, 32, 64, 128, 256])
    b = rng.choice([1, 1, 2, 3, 5, 8, 16, 33, 64])
    hi = _length(rng, 1, 131072 if op == "attend" and b == 1 else 16384)
    n = 1
    if op == "write" or rng.random() < 0.5:
        n = min(hi, _length(rng, 1, 2048))
    new = "one" if b > 1 and rng.random() < 0.3 else "all"
    # At most the largest listed cases' cache, tokens and scores (a plain form holds them padded).
    while b > 1 and (b * hi * hkv * d > 2.0e8 or (op == "write" and b * n > 8192)
                     or (op == "attend" and b * hq * n * hi > 5e8)):
        b //= 2
    while op == "attend" and b * hq * n * hi > 5e8:
        n = max(1, n // 2)
    lo = max(1, n, int(hi * rng.choice([0.1, 0.5, 1.0])))
    if b == 1:
        lo, new = hi, "all"
    return _case("", op, dtype, q8, b, hq, hkv, d, page, min(lo, hi), hi, min(n, hi), new,
                 op == "attend" and rng.random() < 0.2, op == "attend" and rng.random() < 0.3)


def _lens(c):
    """Tokens of each sequence, evenly spread from `hi` down to `lo`."""
    b = c["b"]
    return [c["hi"] - (c["hi"] - c["lo"]) * i // max(1, b - 1) for i in range(b)]


def _news(c):
    """New tokens of each sequence."""
    if c["new"] == "one":
        return [c["n"]] + [1] * (c["b"] - 1)
    return [min(c["n"], x) for x in _lens(c)]


def _gone(c):
    """Leading pages of each sequence that are gone: a quarter of the tokens before the new ones."""
    return [(x - n) // 4 // c["page"] if c["gone"] and i % 2 == 0 else 0
            for i, (x, n) in enumerate(zip(_lens(c), _news(c)))]


# ---- the plain form: elementary operations in 32 bits ------------------------


def _quantise(x, top):
    """e4m3 codes and e8m0 scales of rows: the smallest power of two (from 2^-126 to 2^top) with
    which no finite value passes 448, larger ones held at it; infinities and NaN are stored as NaN."""
    x = x.float()
    fine = torch.isfinite(x)
    amax = torch.where(fine, x, 0.0).abs().amax(-1)
    f, k = torch.frexp(amax)
    e = torch.where(f <= 0.875, k - 9, k - 8)
    e = torch.where(amax == 0, -126, e).clamp(-126, top)
    y = torch.ldexp(x, -e[..., None]).clamp(-448, 448)
    y = torch.where(fine, y, math.nan)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _row_of(s):
    """(sequence, position) of every new token's row."""
    t = s["k_new"].shape[0] if s["k_new"] is not None else s["q"].shape[0]
    row = torch.arange(t, device=s["seq_lens"].device)
    seq = torch.searchsorted(s["cu"][1:], row, right=True)
    return seq, s["seq_lens"][seq] - s["cu"][1:][seq] + row


def _plain_write(s):
    page = s["k"].shape[2]
    seq, pos = _row_of(s)
    at = (s["table"][seq, pos // page].long(), slice(None), pos % page)
    for pool, scale, new in ((s["k"], s["ks"], s["k_new"]), (s["v"], s["vs"], s["v_new"])):
        if scale is None:
            pool[at] = new
        else:
            pool[at], scale[at] = _quantise(new, s["top"])


def _gathered(s, longest):
    """K and V in 32 bits, [B, Hkv, longest, D] with zeros past a sequence's end and in pages that are
    gone, and which of the positions hold a token, [B, longest]."""
    page = s["k"].shape[2]
    pos = torch.arange(longest, device=s["k"].device)
    pages = s["table"][:, pos // page].long()
    held = (pos < s["seq_lens"][:, None]) & (pages >= 0)
    at = (pages.clamp(min=0), slice(None), (pos % page).expand_as(pages))
    got = []
    for pool, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        x = pool[at].float()  # [B, longest, Hkv, D]
        if scale is not None:
            x = x * scale[at].float()[..., None]
        got.append(torch.where(held[:, :, None, None], x, 0.0).transpose(1, 2).contiguous())
    return got[0], got[1], held


def _plain_attend(s):
    c, q = s["case"], s["q"]
    b, hq, hkv, d = c["b"], c["hq"], c["hkv"], c["d"]
    k, v, held = _gathered(s, s["longest"])
    n = s["most_new"]
    seq, pos = _row_of(s)
    col = pos - (s["seq_lens"] - s["cu"].diff())[seq]
    qp = torch.zeros(b, n, hq, d, device=q.device)
    qp[seq, col] = q.float()
    at = torch.zeros(b, n, dtype=torch.long, device=q.device)
    at[seq, col] = pos.long()
    seen = held[:, None, :] & (torch.arange(k.shape[2], device=q.device) <= at[:, :, None])
    seen = seen[:, None, None]  # [B, 1, 1, n, longest]
    qp = qp.view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    x = (qp @ k.transpose(2, 3).contiguous() * s["scale"]).view(b, hkv, hq // hkv, n, -1)
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hkv, -1, k.shape[2]) @ v).view(b, hkv, hq // hkv, n, d)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)[seq, col].to(q.dtype)
    if not c["lse"]:
        return o
    lse = (m + torch.log(total)).permute(1, 2, 0, 3, 4).reshape(hq, b, n)[:, seq, col]
    return o, lse


# ---- what is measured -----------------------------------------------------------


def prepare(c, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dev, dt = "cuda", DTYPES[c["dtype"]]
    b, hq, hkv, d, page = (c[x] for x in ("b", "hq", "hkv", "d", "page"))
    order = torch.randperm(b - 1, device=dev, generator=g) + 1 if b > 1 else None
    lens, news, gone = (torch.tensor(f(c), device=dev, dtype=torch.int32) for f in (_lens, _news, _gone))
    if b > 1:  # the batch in any order behind its first sequence
        order = torch.cat([order.new_zeros(1), order])
        lens, news, gone = lens[order], news[order], gone[order]
    need = [-(-x // page) for x in _lens(c)]
    width = max(need)
    pool = sum(need) + 4
    # Each sequence's pages, from anywhere in the pool; entries behind them are unused.
    col = torch.arange(width, device=dev)
    used = col < ((lens + page - 1) // page)[:, None]
    table = torch.full((b, width), -1, dtype=torch.int32, device=dev)
    table[used] = torch.randperm(pool, device=dev, generator=g)[: sum(need)].int()
    table[col < gone[:, None]] = -1
    cu = torch.zeros(b + 1, dtype=torch.int32, device=dev)
    cu[1:] = news.cumsum(0)
    t = sum(_news(c))

    def rows(*shape):  # tokens whose size varies, as a projection gives them
        size = torch.exp(0.5 * torch.randn(*shape[:-1], 1, device=dev, generator=g))
        return (torch.randn(*shape, device=dev, dtype=dt, generator=g) * size.to(dt))

    s = {"case": c, "table": table, "seq_lens": lens, "cu": cu, "longest": c["hi"],
         "most_new": max(_news(c)), "top": TOP[c["dtype"]], "scale": 1.0 / math.sqrt(d), "dtype": dt,
         "q": None, "k_new": None, "v_new": None}
    for x in "kv":
        s[x], s[x + "s"] = rows(pool, hkv, page, d), None
        if c["q8"]:
            s[x], s[x + "s"] = _quantise(s[x], s["top"])
    if c["op"] == "write":  # K and V as views of one projection's output
        s["k_new"], s["v_new"] = rows(t, 2, hkv, d).unbind(1)
    if c["op"] == "attend":
        s["q"] = torch.randn(t, hq, d, device=dev, dtype=dt, generator=g)
    return s


def run(s):
    c = s["case"]
    scales = {"k_scale": s["ks"], "v_scale": s["vs"]}
    paged = (s["k"], s["v"], s["table"], s["seq_lens"])
    cu = None if s["most_new"] == 1 else s["cu"]  # one new token in every sequence
    if c["op"] == "write":
        if own:
            _fa().paged_cache_write(s["k_new"], s["v_new"], *paged, cu_seqlens=cu, **scales)
        else:
            _plain_write(s)
        return [x for x in (s["k"], s["v"], s["ks"], s["vs"]) if x is not None]
    if c["op"] == "read":
        if own:
            return _fa().paged_cache_read(*paged, max_len=s["longest"], dtype=s["dtype"], **scales)
        k, v, _ = _gathered(s, s["longest"])
        return k.to(s["dtype"]), v.to(s["dtype"])
    if own:
        return _fa().flash_attention_paged(s["q"], *paged, cu_seqlens=cu, max_query_len=s["most_new"],
                                           return_lse=c["lse"], **scales)
    return _plain_attend(s)


def _pairs(c):
    """(new token, key) pairs that take part, over the batch, for one head."""
    return sum(n * (x - n) + n * (n + 1) // 2 - n * g * c["page"]
               for x, n, g in zip(_lens(c), _news(c), _gone(c)))


def work(c):
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    held = sum(x - g * c["page"] for x, g in zip(_lens(c), _gone(c)))
    t = sum(_news(c))
    row = 2 * hkv * (d + 1 if c["q8"] else 2 * d)  # one token's K and V in the cache
    pages = sum(-(-x // c["page"]) for x in _lens(c))
    if c["op"] == "write":
        return {"bytes": t * (2 * hkv * 2 * d + row) + 12 * c["b"], "flops": 0}
    if c["op"] == "read":
        return {"bytes": held * row + c["b"] * c["hi"] * 2 * hkv * 2 * d + 4 * pages, "flops": 0}
    return {"bytes": 2 * t * hq * 2 * d + held * row + 4 * pages + (4 * t * hq if c["lse"] else 0),
            "flops": 4 * hq * d * _pairs(c)}


# ---- the definition in 64 bits --------------------------------------------------


def _e4m3(x, top):
    """Rows of 64-bit values as the quantised values' codes and scales, by arithmetic."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 448))
    e = torch.where(448 * torch.exp2(e - 1) >= amax, e - 1, e)
    e = torch.where(448 * torch.exp2(e) < amax, e + 1, e)
    scale = torch.exp2(e.clamp(-126, top))
    y = (x / scale).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, scale[..., 0]


def exact(c, seed):
    s = prepare(c, seed)
    lens, cu, table = s["seq_lens"].tolist(), s["cu"].tolist(), s["table"].tolist()
    page, hq, hkv, d, dev = c["page"], c["hq"], c["hkv"], c["d"], s["table"].device
    if c["op"] == "write":
        out = []
        for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
            pool, new = pool.double(), new.double()
            scale = None
            if c["q8"]:
                scale = (s["ks"] if not out else s["vs"]).double()
                new, new_scale = _e4m3(new, s["top"])
            for i in range(c["b"]):
                n = cu[i + 1] - cu[i]
                at = list(range(lens[i] - n, lens[i]))
                to = torch.tensor([table[i][p // page] for p in at], device=dev)
                off = torch.tensor([p % page for p in at], device=dev)
                pool[to, :, off] = new[cu[i]:cu[i + 1]]
                if scale is not None:
                    scale[to, :, off] = new_scale[cu[i]:cu[i + 1]]
            out.append((pool, scale))
        return [x for x in (out[0][0], out[1][0], out[0][1], out[1][1]) if x is not None]

    def cached(i, pool, scale):
        """Sequence i's rows that it still holds, [Hkv, rows, D], and their positions."""
        pages = [(j, p) for j, p in enumerate(table[i][: -(-lens[i] // page)]) if p >= 0]
        at = torch.tensor([j for j, _ in pages], device=dev)[:, None] * page + torch.arange(page, device=dev)
        ids = torch.tensor([p for _, p in pages], device=dev)
        x = pool[ids].double()
        if scale is not None:
            x = x * scale[ids].double()[..., None]
        x, at = x.transpose(0, 1).reshape(hkv, -1, d), at.reshape(-1)
        return x[:, at < lens[i]], at[at < lens[i]]

    if c["op"] == "read":
        got = []
        for x in "kv":
            y = torch.zeros(c["b"], hkv, c["hi"], d, dtype=torch.float64, device=dev)
            for i in range(c["b"]):
                z, at = cached(i, s[x], s[x + "s"])
                y[i][:, at] = z
            got.append(y)
        return tuple(got)
    o = torch.zeros(cu[-1], hq, d, dtype=torch.float64, device=dev)
    lse = torch.zeros(hq, cu[-1], dtype=torch.float64, device=dev)
    for i in range(c["b"]):
        (k, at), (v, _) = cached(i, s["k"], s["ks"]), cached(i, s["v"], s["vs"])
        n = cu[i + 1] - cu[i]
        hidden = at[None, :] > torch.arange(lens[i] - n, lens[i], device=dev)[:, None]
        for h in range(hq):
            g = h // (hq // hkv)
            x = s["q"][cu[i]:cu[i + 1], h].double() @ k[g].t() * s["scale"]
            x.masked_fill_(hidden, -math.inf)
            row = torch.logsumexp(x, -1)
            lse[h, cu[i]:cu[i + 1]] = row
            o[cu[i]:cu[i + 1], h] = torch.exp(x - row[:, None]) @ v[g]
    return (o, lse) if c["lse"] else o
