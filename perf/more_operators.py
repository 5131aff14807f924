"""Timing cases of what a server does with long contexts in the paged key/value cache: attention of
sequences that share a prefix, the weight that attention gave each cached row, and eviction by it.

A cache is a pool of pages, [pages, heads_kv, page_size, head_dim] for K and the same for V, in the
model's 16-bit type or in 8 bits (e4m3 codes, and a power-of-two scale for each token and head, e8m0).
`block_table[b]` lists the pages of sequence b in order, a negative entry being a page that is gone;
`seq_lens[b]` counts its tokens, the new ones included, which are its last ones;
`cu_seqlens[b] .. cu_seqlens[b + 1]` are their rows in Q ([tokens, heads, head_dim]).

  prefix  flash_attention_paged_prefix: softmax(scale Q K^T) V where sequences cu_prefix[g] ..
          cu_prefix[g + 1] - 1 see all of prefix g (prefix_table[g], prefix_lens[g]), then their own rows:
          token i of n own keys 0 .. seq_len - n + i; sequences behind the last group have no prefix
  weigh   paged_attention_weights: for each cached row of a KV head, the sum of the probabilities
          exp(scale q k - LSE) that the new tokens' query heads of its group gave it
  evict   paged_cache_evict: of each sequence and KV head the rows of the last `recent` positions and
          the heaviest others, `keep` in all, copied in order to the pages of another table, with
          their weights
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# The largest scale of an 8-bit row: 448 times it is finite in the rows' type.
TOP = {"fp16": 7, "bf16": 119}


def _fa():
    """The package, imported once, where its calls are the ones that run."""
    if not hasattr(_fa, "package"):
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "flash-attention-sm75-register-fused_amd", "src"))
        import flash_attention_sm75

        _fa.package = flash_attention_sm75
    return _fa.package


def _case(name, op, dtype, q8, b, hq, hkv, d, page, lo, hi, n=1, prefix=0, groups=1, alone=0, lse=False,
          gone=False, keep=0, recent=0):
    """`b` sequences of `lo` to `hi` own tokens, the last `n` of them new; prefix: `groups` prefixes of
    up to `prefix` tokens, of which the last `alone` sequences have none; evict: `keep` rows stay, those
    of the last `recent` positions among them; gone: the first pages of every other sequence are."""
    c = {"op": op, "dtype": dtype, "q8": q8, "b": b, "hq": hq, "hkv": hkv, "d": d, "page": page,
         "lo": lo, "hi": hi, "n": n, "prefix": prefix, "groups": groups, "alone": alone, "lse": lse,
         "gone": gone, "keep": keep, "recent": recent}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token each of a few answers to one prompt: once per layer and token, latency counts
        _case("prefix_token", "prefix", "bf16", False, 4, 14, 2, 64, 16, 17, 60, prefix=1000),
        # one token of each request of a serving batch behind a long common instruction
        _case("prefix_batch", "prefix", "fp16", False, 64, 32, 8, 128, 64, 128, 1024, prefix=8192),
        # several documents, each with its own readers, some requests without, in 8 bits
        _case("prefix_groups_q8", "prefix", "bf16", True, 48, 32, 8, 128, 32, 100, 1500, prefix=16384,
              groups=5, alone=3),
        # questions to one document arrive together: their prompts behind it, log-sum-exp kept to weigh rows
        _case("prefix_questions", "prefix", "bf16", False, 13, 32, 8, 128, 64, 61, 250, n=250, prefix=8192,
              lse=True),
        # the weights of one generated token: once per layer and token, latency counts
        _case("weigh_token", "weigh", "bf16", False, 1, 14, 2, 64, 16, 4097, 4097),
        # those of a serving batch's tokens over 8 bits: streaming K
        _case("weigh_batch_q8", "weigh", "fp16", True, 32, 32, 8, 128, 32, 4096, 8192),
        # a prompt's last tokens weigh the rows before them, odd lengths, early pages gone
        _case("weigh_window", "weigh", "fp16", False, 5, 14, 2, 64, 16, 3001, 16000, n=33, gone=True),
        # every token of a long prompt's later chunk: the largest product
        _case("weigh_chunk", "weigh", "bf16", False, 1, 32, 8, 128, 64, 8192, 8192, n=2048),
        # a short conversation is cut to half: latency counts
        _case("evict_one", "evict", "bf16", False, 1, 14, 2, 64, 16, 1025, 1025, keep=512, recent=32),
        # a serving batch's sequences are cut to one length
        _case("evict_batch", "evict", "fp16", False, 32, 32, 8, 128, 64, 4096, 8192, keep=2048, recent=256),
        # the same in 8 bits, odd numbers, some shorter than what is kept, early pages gone
        _case("evict_ragged_q8", "evict", "bf16", True, 24, 12, 12, 64, 16, 333, 5555, keep=1501, recent=99,
              gone=True),
        # one very long context
        _case("evict_long", "evict", "bf16", False, 1, 32, 8, 128, 128, 131072, 131072, keep=16384, recent=1024),
    ]


# (query heads, KV heads, head_dim) of the repository's configurations, tests and benchmark
HEADS = [(1, 1, 64), (8, 8, 64), (8, 8, 128), (12, 12, 64), (14, 2, 64), (16, 4, 128), (32, 8, 64),
         (32, 8, 128), (64, 8, 128)]


def _length(rng, lo, hi):
    """Spread over the logarithm; one in four a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(64, n // 64 * 64) if hi >= 64 and rng.random() < 1 / 4 else n


def draw(rng):
    op = rng.choice(["prefix", "prefix", "weigh", "evict"])
    hq, hkv, d = rng.choice(HEADS)
    dtype, q8 = rng.choice(["fp16", "bf16"]), rng.random() < 0.5
    page = rng.choice([16, 16, 32, 64, 128, 256])
    b = rng.choice([1, 1, 2, 3, 5, 8, 16, 33, 64])
    if op == "evict":
        hi = _length(rng, 2, 131072 if b == 1 else 16384)
        while b > 1 and b * hi * hkv * d > 2.0e8:
            b //= 2
        lo = hi if b == 1 else max(1, int(hi * rng.choice([0.1, 0.5, 1.0])))
        keep = max(1, int(hi * rng.uniform(0.1, 0.8)))
        return _case("", op, dtype, q8, b, hq, hkv, d, page, lo, hi, gone=rng.random() < 0.2, keep=keep,
                     recent=min(keep, int(keep * rng.choice([0.0, 0.1, 0.5]))))
    if op == "weigh":
        hi = _length(rng, 1, 65536 if b == 1 else 16384)
        n = min(hi, _length(rng, 1, 2048)) if rng.random() < 0.5 else 1
        # At most the largest listed cases' cache and scores (a plain form holds them padded).
        while b > 1 and (b * hi * hkv * d > 2.0e8 or b * hq * n * hi > 5e8):
            b //= 2
        while b * hq * n * hi > 5e8:
            n = max(1, n // 2)
        lo = hi if b == 1 else max(n, int(hi * rng.choice([0.1, 0.5, 1.0])), 1)
        return _case("", op, dtype, q8, b, hq, hkv, d, page, lo, hi, n=n, gone=rng.random() < 0.2)
    b = max(2, b)
    prefix, hi = _length(rng, 1, 16384), _length(rng, 1, 2048)
    n = min(hi, _length(rng, 1, 512)) if rng.random() < 0.4 else 1
    while b > 2 and b * hi * hkv * d > 1.0e8:
        b //= 2
    while b * n * hq * (prefix + hi) > 1e9 and n > 1:
        n = max(1, n // 2)
    groups = rng.choice([1, 1, 2, 3, 5])
    alone = rng.choice([0, 0, 1])
    groups = max(1, min(groups, b - alone))
    return _case("", op, dtype, q8, b, hq, hkv, d, page, max(n, int(hi * rng.choice([0.1, 0.5, 1.0])), 1), hi,
                 n=n, prefix=prefix, groups=groups, alone=alone, lse=rng.random() < 0.3)


def _lens(c):
    """Own tokens of each sequence, evenly spread from `hi` down to `lo`."""
    b = c["b"]
    return [c["hi"] - (c["hi"] - c["lo"]) * i // max(1, b - 1) for i in range(b)]


def _news(c):
    return [min(c["n"], x) for x in _lens(c)]


def _gone(c):
    """Leading pages of each sequence that are gone: a quarter of the tokens before the new ones."""
    return [(x - n) // 4 // c["page"] if c["gone"] and i % 2 == 0 else 0
            for i, (x, n) in enumerate(zip(_lens(c), _news(c)))]


def _prefixes(c):
    """Tokens of each prefix, from `prefix` down to a third of it."""
    g = c["groups"]
    return [max(1, c["prefix"] - c["prefix"] * 2 * i // (3 * max(1, g - 1))) for i in range(g)]


def _cu_prefix(c):
    """Where each prefix's sequences begin; behind the last they have none."""
    g, b = c["groups"], c["b"] - c["alone"]
    return [b * i // g for i in range(g + 1)]


# ---- the plain form: elementary operations in 32 bits ------------------------


def _quantise(x, top):
    """e4m3 codes and e8m0 scales of rows: the smallest power of two (from 2^-126 to 2^top) with
    which no finite value passes 448."""
    x = x.float()
    f, k = torch.frexp(x.abs().amax(-1))
    e = torch.where(f <= 0.875, k - 9, k - 8).clamp(-126, top)
    y = torch.ldexp(x, -e[..., None]).clamp(-448, 448)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _row_of(s):
    """(sequence, position) of every new token's row."""
    row = torch.arange(s["q"].shape[0], device=s["seq_lens"].device)
    seq = torch.searchsorted(s["cu"][1:], row, right=True)
    return seq, s["seq_lens"][seq] - s["cu"][1:][seq] + row


def _gathered(s, table, lens, longest, pools="kv"):
    """K and V (or those of `pools`) of a table's rows in 32 bits, [B, Hkv, longest, D] with zeros where
    there is no token, and which of the positions hold one, [B, longest]."""
    page = s["k"].shape[2]
    pos = torch.arange(longest, device=s["k"].device)
    pages = table[:, pos // page].long()
    held = (pos < lens[:, None]) & (pages >= 0)
    at = (pages.clamp(min=0), slice(None), (pos % page).expand_as(pages))
    got = []
    for x in pools:
        y = s[x][at].float()  # [B, longest, Hkv, D]
        if s[x + "s"] is not None:
            y = y * s[x + "s"][at].float()[..., None]
        got.append(torch.where(held[:, :, None, None], y, 0.0).transpose(1, 2).contiguous())
    return *got, held


def _padded(s):
    """Q padded to [B, Hkv, group * n, D], and which (row, key) pairs of the sequences' own rows there are."""
    c, q = s["case"], s["q"]
    b, hq, hkv, d, n = c["b"], c["hq"], c["hkv"], c["d"], max(_news(s["case"]))
    seq, pos = _row_of(s)
    col = pos - (s["seq_lens"] - s["cu"].diff())[seq]
    qp = torch.zeros(b, n, hq, d, device=q.device)
    qp[seq, col] = q.float()
    at = torch.full((b, n), -1, dtype=torch.long, device=q.device)
    at[seq, col] = pos.long()
    qp = qp.view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    return qp, at, seq, col


def _scores(s, k, held, qp, at):
    """Scores of the padded rows and their own keys, [B, Hkv, group, n, keys], -inf where hidden."""
    b, hkv, n = k.shape[0], k.shape[1], at.shape[1]
    seen = held[:, None, :] & (torch.arange(k.shape[2], device=k.device) <= at[:, :, None])
    x = (qp @ k.transpose(2, 3).contiguous() * s["scale"]).view(b, hkv, -1, n, k.shape[2])
    return torch.where(seen[:, None, None], x, -math.inf)


def _state(x, v):
    """Running maximum, sum and weighted sum of V of scores [..., rows, keys]."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    return m, p.sum(-1, keepdim=True), p @ v


def _plain_prefix(s):
    c, q = s["case"], s["q"]
    b, hq, hkv, d = c["b"], c["hq"], c["hkv"], c["d"]
    k, v, held = _gathered(s, s["table"], s["seq_lens"], c["hi"])
    qp, at, seq, col = _padded(s)
    n = at.shape[1]
    x = _scores(s, k, held, qp, at).view(b, hkv, -1, c["hi"])
    m, l, o = _state(x, v)
    cu, lens = _cu_prefix(c), _prefixes(c)
    for g in range(c["groups"]):  # the prefix's rows once for all of its sequences
        pk, pv, _ = _gathered(s, s["prefix_table"][g:g + 1], s["prefix_lens"][g:g + 1], lens[g])
        rows = slice(cu[g], cu[g + 1])
        y = qp[rows].transpose(0, 1).reshape(hkv, -1, d) @ pk[0].transpose(1, 2).contiguous() * s["scale"]
        mp, lp, op = (z.view(hkv, cu[g + 1] - cu[g], -1, z.shape[-1]).transpose(0, 1) for z in _state(y, pv[0]))
        top = torch.maximum(m[rows], mp)
        f, fp = torch.exp(m[rows] - top), torch.exp(mp - top)
        l[rows], o[rows] = f * l[rows] + fp * lp, f * o[rows] + fp * op
        m[rows] = top
    o = torch.where(l > 0, o / l, 0.0).view(b, hkv, hq // hkv, n, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)[seq, col].to(q.dtype)
    if not c["lse"]:
        return o
    return o, (m + torch.log(l)).view(b, hkv, -1, n).permute(1, 2, 0, 3).reshape(hq, b, n)[:, seq, col]


def _plain_weigh(s):
    c, lse = s["case"], s["lse"]
    k, held = _gathered(s, s["table"], s["seq_lens"], s["room"], "k")
    qp, at, seq, col = _padded(s)
    z = torch.full((c["hq"], c["b"], at.shape[1]), math.inf, device=lse.device)
    z[:, seq, col] = lse
    z = z.view(c["hkv"], -1, c["b"], at.shape[1]).permute(2, 0, 1, 3)
    return torch.exp(_scores(s, k, held, qp, at) - z[..., None]).sum((2, 3))


def _plain_evict(s):
    c, w = s["case"], s["weights"]
    page, keep = c["page"], c["keep"]
    pos = torch.arange(s["room"], device=w.device)
    pages = s["table"][:, pos // page].long()
    held = (pos < s["seq_lens"][:, None]) & (pages >= 0)
    recent = pos >= s["seq_lens"][:, None] - c["recent"]
    rank = torch.where(held[:, None], torch.where(recent[:, None], math.inf, w), -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    lens = held.sum(-1).clamp(max=keep)
    here = torch.arange(order.shape[-1], device=w.device) < lens[:, None]  # rows that stay, [B, keep]
    order = torch.where(here[:, None], order, s["room"]).sort(-1).values
    b, r = here.nonzero(as_tuple=True)
    src = order[b, :, r]  # [rows, Hkv]
    h = torch.arange(c["hkv"], device=w.device)
    kept = torch.zeros(c["b"], c["hkv"], s["to_table"].shape[1] * page, device=w.device)
    kept[b[:, None], h, r[:, None]] = w[b[:, None], h, src]
    at = (pages[b[:, None], src], h, src % page)
    to = (s["to_table"][b, r // page].long()[:, None], h, (r % page)[:, None])
    for x in ("k", "v", "ks", "vs"):
        if s[x] is not None:
            s[x][to] = s[x][at]
    return lens.int(), kept


# ---- what is measured -----------------------------------------------------------


def _table(need, width, ids, device):
    """Rows of page numbers, need[i] of them taken from `ids`, -1 behind."""
    t = torch.full((len(need), width), -1, dtype=torch.int32, device=device)
    col = torch.arange(width, device=device)
    used = col < torch.tensor(need, device=device)[:, None]
    t[used] = ids[: sum(need)]
    return t


def prepare(c, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dev, dt = "cuda", DTYPES[c["dtype"]]
    b, hq, hkv, d, page = (c[x] for x in ("b", "hq", "hkv", "d", "page"))
    lens, news, gone = _lens(c), _news(c), _gone(c)
    need = [-(-x // page) for x in lens]
    prefixes = _prefixes(c) if c["op"] == "prefix" else []
    pneed = [-(-x // page) for x in prefixes]
    kneed = [-(-(c["keep"] + 1) // page)] * b if c["op"] == "evict" else []  # room for the next token
    # Every table's pages, from anywhere in the pool; entries behind them are unused.
    pool = sum(need) + sum(pneed) + sum(kneed) + 4
    ids = torch.randperm(pool, device=dev, generator=g).int()
    table = _table(need, max(need), ids, dev)
    table[torch.arange(max(need), device=dev) < torch.tensor(gone, device=dev)[:, None]] = -1
    cu = torch.tensor([0] + news, device=dev).cumsum(0).int()

    def rows(*shape):  # tokens whose size varies, as a projection gives them
        size = torch.exp(0.5 * torch.randn(*shape[:-1], 1, device=dev, generator=g))
        return torch.randn(*shape, device=dev, dtype=dt, generator=g) * size.to(dt)

    s = {"case": c, "table": table, "seq_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "cu": cu,
         "scale": 1.0 / math.sqrt(d), "room": max(need) * page}
    for x in "kv":
        s[x], s[x + "s"] = rows(pool, hkv, page, d), None
        if c["q8"]:
            s[x], s[x + "s"] = _quantise(s[x], TOP[c["dtype"]])
    if c["op"] != "evict":
        s["q"] = torch.randn(sum(news), hq, d, device=dev, dtype=dt, generator=g)
    if c["op"] == "prefix":
        s["prefix_table"] = _table(pneed, max(pneed), ids[sum(need):], dev)
        s["prefix_lens"] = torch.tensor(prefixes, dtype=torch.int32, device=dev)
        s["cu_prefix"] = torch.tensor(_cu_prefix(c), dtype=torch.int32, device=dev)
        bounds = [0] + torch.tensor(news).cumsum(0).tolist()
        at = _cu_prefix(c)
        s["most_shared"] = max(bounds[at[i + 1]] - bounds[at[i]] for i in range(c["groups"]))
    if c["op"] == "weigh":  # the log-sum-exp of the attention that these tokens had
        k, held = _gathered(s, table, s["seq_lens"], s["room"], "k")
        qp, at, seq, col = _padded(s)
        z = torch.logsumexp(_scores(s, k, held, qp, at), -1)
        s["lse"] = z.permute(1, 2, 0, 3).reshape(hq, b, -1)[:, seq, col].contiguous()
    if c["op"] == "evict":  # sums of probabilities: a few rows have most of it, early ones more
        s["to_table"] = _table(kneed, kneed[0], ids[sum(need):], dev)
        pos = torch.arange(s["room"], device=dev)
        w = torch.exp(2.0 * torch.randn(b, hkv, s["room"], device=dev, generator=g)) / (1.0 + 0.01 * pos)
        s["weights"] = torch.where(pos < s["seq_lens"][:, None, None], w, 0.0)
    return s


def run(s):
    c = s["case"]
    one = c["n"] == 1  # one new token in every sequence
    if c["op"] == "evict":
        if own:
            lens, kept = _fa().paged_cache_evict(s["k"], s["v"], s["table"], s["seq_lens"], s["weights"],
                                                 s["to_table"], c["keep"], recent=c["recent"], k_scale=s["ks"],
                                                 v_scale=s["vs"])
        else:
            lens, kept = _plain_evict(s)
        return [lens, kept] + [s[x] for x in ("k", "v", "ks", "vs") if s[x] is not None]
    if c["op"] == "weigh":
        if own:
            return _fa().paged_attention_weights(s["q"], s["lse"], s["k"], s["table"], s["seq_lens"],
                                                 cu_seqlens=None if one else s["cu"], max_query_len=c["n"],
                                                 k_scale=s["ks"])
        return _plain_weigh(s)
    if own:
        every = c["groups"] == 1 and c["alone"] == 0  # one prefix for the whole batch
        return _fa().flash_attention_paged_prefix(
            s["q"], s["k"], s["v"], s["prefix_table"], s["prefix_lens"], s["table"], s["seq_lens"],
            cu_seqlens=None if one else s["cu"], cu_prefix=None if every else s["cu_prefix"],
            max_query_len=c["n"], max_prefix_queries=s["most_shared"], k_scale=s["ks"], v_scale=s["vs"],
            return_lse=c["lse"])
    return _plain_prefix(s)


def _pairs(c):
    """(new token, own key) pairs that take part, over the batch, for one head."""
    return sum(n * (x - n) + n * (n + 1) // 2 - n * g * c["page"]
               for x, n, g in zip(_lens(c), _news(c), _gone(c)))


def work(c):
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    held = [x - g * page for x, g in zip(_lens(c), _gone(c))]
    row = hkv * (d + 1 if c["q8"] else 2 * d)  # one token's K (or V) in the cache
    t, pages = sum(_news(c)), sum(-(-x // page) for x in _lens(c))
    if c["op"] == "evict":
        kept = sum(min(x, c["keep"]) for x in held)
        room = c["b"] * -(-(c["keep"] + 1) // page) * page
        return {"bytes": 4 * hkv * (sum(held) + room) + 4 * kept * row + 4 * pages, "flops": 0}
    if c["op"] == "weigh":
        room = c["b"] * -(-c["hi"] // page) * page
        return {"bytes": t * hq * (2 * d + 4) + sum(held) * row + 4 * room * hkv + 4 * pages,
                "flops": 2 * hq * d * _pairs(c)}
    prefixes, cu = _prefixes(c), _cu_prefix(c)
    shared = sum(p * sum(_news(c)[cu[i]:cu[i + 1]]) for i, p in enumerate(prefixes))
    return {"bytes": 2 * t * hq * 2 * d + 2 * (sum(held) + sum(prefixes)) * row + 4 * pages
            + (4 * t * hq if c["lse"] else 0),
            "flops": 4 * hq * d * (_pairs(c) + shared)}


# ---- the definition in 64 bits --------------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    lens, cu, table = s["seq_lens"].tolist(), s["cu"].tolist(), s["table"].tolist()
    page, hq, hkv, dev = c["page"], c["hq"], c["hkv"], s["table"].device

    def cached(entries, length, x):
        """A sequence's rows that are held, [Hkv, rows, D], and their positions."""
        pages = [(j, p) for j, p in enumerate(entries[: -(-length // page)]) if p >= 0]
        at = torch.tensor([j for j, _ in pages], device=dev)[:, None] * page + torch.arange(page, device=dev)
        ids = torch.tensor([p for _, p in pages], device=dev)
        y = s[x][ids].double()
        if s[x + "s"] is not None:
            y = y * s[x + "s"][ids].double()[..., None]
        y, at = y.transpose(0, 1).reshape(hkv, -1, c["d"]), at.reshape(-1)
        return y[:, at < length], at[at < length]

    if c["op"] == "evict":
        out = {x: s[x].double() for x in ("k", "v", "ks", "vs") if s[x] is not None}
        kept = torch.zeros(c["b"], hkv, s["to_table"].shape[1] * page, dtype=torch.float64, device=dev)
        left = []
        for i in range(c["b"]):
            pos = torch.arange(lens[i], device=dev)
            ids = s["table"][i][pos // page].long()
            pos, ids = pos[ids >= 0], ids[ids >= 0]
            left.append(min(c["keep"], len(pos)))
            to = s["to_table"][i].long()[torch.arange(left[i], device=dev) // page]
            off = torch.arange(left[i], device=dev) % page
            for h in range(hkv):
                w = s["weights"][i, h].double()[pos]
                stays = pos >= lens[i] - c["recent"]
                more = left[i] - int(stays.sum())
                if more > 0:  # all above the value that bounds them, then the first that equal it
                    rest = w[~stays]
                    bound = torch.kthvalue(rest, len(rest) - more + 1).values
                    above, equal = ~stays & (w > bound), ~stays & (w == bound)
                    equal &= equal.cumsum(0) <= more - int(above.sum())
                    stays = stays | above | equal
                for x, y in out.items():
                    y[to, h, off] = s[x][ids[stays], h, pos[stays] % page].double()
                kept[i, h, : left[i]] = w[stays]
        return [torch.tensor(left, dtype=torch.int32, device=dev), kept] + list(out.values())

    if c["op"] == "weigh":
        w = torch.zeros(c["b"], hkv, s["room"], dtype=torch.float64, device=dev)
        for i in range(c["b"]):
            k, at = cached(table[i], lens[i], "k")
            n = cu[i + 1] - cu[i]
            hidden = at[None, :] > torch.arange(lens[i] - n, lens[i], device=dev)[:, None]
            for h in range(hq):
                x = s["q"][cu[i]:cu[i + 1], h].double() @ k[h // (hq // hkv)].t() * s["scale"]
                p = torch.exp(x - s["lse"][h, cu[i]:cu[i + 1], None].double()).masked_fill(hidden, 0.0)
                w[i, h // (hq // hkv), at] += p.sum(0)
        return w

    o = torch.zeros(cu[-1], hq, c["d"], dtype=torch.float64, device=dev)
    lse = torch.zeros(hq, cu[-1], dtype=torch.float64, device=dev)
    first, last = _cu_prefix(c), -1
    for i in range(c["b"]):
        (k, at), (v, _) = cached(table[i], lens[i], "k"), cached(table[i], lens[i], "v")
        n = cu[i + 1] - cu[i]
        hidden = at[None, :] > torch.arange(lens[i] - n, lens[i], device=dev)[:, None]
        g = sum(f <= i for f in first) - 1
        if g < c["groups"]:
            if g != last:
                rows = s["prefix_table"][g].tolist(), int(s["prefix_lens"][g])
                (pk, _), (pv, _), last = cached(*rows, "k"), cached(*rows, "v"), g
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
            hidden = torch.cat([hidden.new_zeros(n, pk.shape[1]), hidden], 1)
        x = s["q"][cu[i]:cu[i + 1]].double().view(n, hkv, -1, c["d"]).permute(1, 2, 0, 3).reshape(hkv, -1, c["d"])
        for h in range(hkv):
            y = (x[h] @ k[h].t() * s["scale"]).view(-1, n, k.shape[1]).masked_fill(hidden, -math.inf)
            z = torch.logsumexp(y, -1)
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            lse[heads, cu[i]:cu[i + 1]] = z
            o[cu[i]:cu[i + 1], heads] = (torch.exp(y - z[..., None]) @ v[h]).transpose(0, 1)
    return (o, lse) if c["lse"] else o
