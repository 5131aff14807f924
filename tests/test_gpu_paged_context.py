"""Long contexts in the paged cache on the GPU against plain 64-bit references: attention behind
shared prefixes, the weights it gave each row, eviction by them, and the three together."""
import math

import pytest
import torch

import flash_attention_sm75 as fa
import paged_context_ref as con
import paged_ref as ref
from paged_ref import Cache

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def groups_of(cu, batch):
    """Sequence b's prefix, or None, from cu_prefix."""
    return [next((g for g in range(len(cu) - 1) if cu[g] <= b < cu[g + 1]), None) for b in range(batch)]


def on(device, own, shared, strided=False):
    """The call's tensors on the device: pools, scales, the prefixes' table and lens, the own ones."""
    pool, table = con.one_pool(own, shared)

    def put(x):
        raw = x.view(torch.uint8) if x.dtype == torch.float8_e8m0fnu else x
        y = raw.transpose(1, 2).contiguous().to(device).transpose(1, 2) if strided else raw.to(device)
        return y.view(x.dtype)
    scales = {"k_scale": put(pool["ks"]), "v_scale": put(pool["vs"])} if own.q8 else {}
    return (put(pool["k"]), put(pool["v"]), table.to(device), shared.seq_lens.to(device), own.table.to(device),
            own.seq_lens.to(device)), scales


def attend(own, shared, cu_prefix, device, hq, seed=1, causal=True, scale=None, strided=False, hints=None, **kw):
    """The call as each of the two kernels takes the prefixes and the own keys, O and LSE checked;
    returns the last."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(own.news), hq, own.d, generator=g).to(own.dtype)
    at = list(range(0, len(own.lens) + 1, len(own.lens))) if cu_prefix is None else cu_prefix
    joined = con.Joined(own, shared, groups_of(at, len(own.lens)))
    want, want_lse, tol, lse_tol = ref.attention(joined, q, causal, scale)
    # Joining two states rounds the weights once more, by 2^-15 of them at most (exp2 of a
    # difference of maxima up to 2^8); tol has 2^-11 of them or more.
    tol, lse_tol = tol * (1 + 2.0 ** -4), lse_tol + 2.0 ** -15
    args, scales = on(device, own, shared, strided)
    ones = all(n == 1 for n in own.news)
    cu_prefix = None if cu_prefix is None else torch.tensor(cu_prefix, dtype=torch.int32, device=device)
    # A table with room for more than 128 MB of prefix rows (one read for each sequence) makes two launches of few rows.
    pools, table, rest = args[:2], args[2], args[3:]
    room = (128 << 20) // (len(own.lens) * own.hkv * 2 * own.d * (1 if own.q8 else 2)) + own.page
    wide = torch.nn.functional.pad(table, (0, max(0, room // own.page + 1 - table.shape[1])), value=-1)
    calls = [(a, b, t) for a, b in hints or ([(None, None), (None, 1)] if ones else
                                             [(1, 1), (1, 10 ** 6), (10 ** 6, 1), (None, None)])
             for t in (table, wide)]
    for own_hint, shared_hint, table in calls:
        o, lse = fa.flash_attention_paged_prefix(
            q.to(device), *pools, table, *rest, cu_seqlens=None if ones else own.cu.to(device), cu_prefix=cu_prefix,
            max_query_len=own_hint, max_prefix_queries=shared_hint, causal="bottom_right" if causal else False,
            scale=scale, return_lse=True, **scales, **kw)
        ref.check(o, want, tol, f"O (hints {own_hint}, {shared_hint}, table {tuple(table.shape)})")
        ref.check(lse, want_lse, lse_tol, f"LSE (hints {own_hint}, {shared_hint}, table {tuple(table.shape)})")
    return o, lse


# ---- shared prefixes -----------------------------------------------------------------


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_prefix_single_tokens(device, d, dtype, q8, page):
    """One token of each sequence; prefixes and own keys around tiles and pages, empty ones among them."""
    own = Cache([1, 0, 15, 16, 17, 33, 64, 65, 130, 300], 2, d, page, dtype, q8)
    shared = Cache([1, 200, 0, 65], 2, d, page, dtype, q8, seed=5)
    attend(own, shared, [0, 1, 4, 6, 9], device, 8)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (14, 2), (12, 12), (32, 8), (15, 3), (40, 2), (16, 16)])
@pytest.mark.parametrize("q8", [False, True])
def test_prefix_heads(device, hq, hkv, q8):
    own, shared = Cache([77, 30, 5, 1], hkv, 64, 16, BF16, q8), Cache([130], hkv, 64, 16, BF16, q8, seed=3)
    attend(own, shared, None, device, hq)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news", [[4, 4, 4], [1, 9, 2], [0, 3, 0], [70, 5, 33], [130, 1, 140]])
@pytest.mark.parametrize("causal", [True, False])
def test_prefix_chunks(device, d, q8, news, causal):
    """Several new tokens a sequence, none in some; own keys may be the new ones alone."""
    lens = [max(n, x) for n, x in zip(news, [90, 20, 140])]
    own, shared = Cache(lens, 2, d, 16, FP16, q8, news=news), Cache([99, 257], 2, d, 16, FP16, q8, seed=4)
    attend(own, shared, [0, 2, 3], device, 6, causal=causal)


@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("q8", [False, True])
def test_prefix_long(device, page, q8):
    """Prefixes split over many workgroups, their rows in several blocks; own keys split too."""
    own = Cache([40, 3, 900, 64, 1] * 7, 2, 128, page, BF16, q8)
    attend(own, Cache([5000, 611], 2, 128, page, BF16, q8, seed=2), [0, 31, 35], device, 8)
    own = Cache([300, 61], 2, 128, page, BF16, q8, news=[40, 61])
    attend(own, Cache([4100], 2, 128, page, BF16, q8, seed=2), None, device, 8)


@pytest.mark.parametrize("d", [64, 128])
def test_prefix_many_blocks(device, d):
    """More units than the GPU runs at once, of the prefix, of the own keys or of both."""
    own = Cache([700, 650], 8, d, 64, BF16, False, news=[700, 300])
    attend(own, Cache([130], 8, d, 64, BF16, False, seed=2), None, device, 32, hints=[(700, None)])


def test_prefix_many_sequences(device):
    """More sequences and prefixes than a wave has lanes."""
    lens = [(7 * i) % 50 for i in range(150)]
    own, shared = Cache(lens, 1, 64, 16, FP16, False), Cache([(11 * i) % 90 for i in range(70)], 1, 64, 16, FP16, False, seed=3)
    attend(own, shared, [2 * i for i in range(71)], device, 4)


def test_prefix_of_some(device):
    """Sequences before the first and behind the last group have none; groups may be empty."""
    own, shared = Cache([40, 50, 60, 33, 20], 2, 64, 16, FP16, True), Cache([100, 7, 64], 2, 64, 16, FP16, True, seed=3)
    attend(own, shared, [1, 3, 3, 4], device, 4)
    attend(own, shared, [5, 5, 5, 5], device, 4)
    attend(own, shared, [0, 0, 0, 0], device, 4)


@pytest.mark.parametrize("sequences,prefixes", [(64, 63), (64, 64), (65, 63)])
def test_prefix_most_in_one_launch(device, sequences, prefixes):
    """Up to 64 sequences and 63 prefixes a few rows' prefixes and own keys are one launch."""
    own = Cache([(5 * i) % 40 for i in range(sequences)], 1, 64, 16, BF16, False, news=[1] * sequences)
    shared = Cache([(7 * i) % 71 for i in range(prefixes)], 1, 64, 16, BF16, False, seed=3)
    attend(own, shared, [min(i + 1, sequences - 1) for i in range(prefixes)] + [sequences - 1], device, 4)


@pytest.mark.parametrize("q8", [False, True])
def test_prefix_tables_without_columns(device, q8):
    """No page of a sequence's own, or none of a prefix's."""
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).half()
    for lens, plens in (([0, 0, 0], [77, 0]), ([40, 0, 33], [0, 0]), ([0, 0, 0], [0, 0])):
        own, shared = Cache(lens, 2, 64, 16, FP16, q8, news=[1, 1, 1]), Cache(plens, 2, 64, 16, FP16, q8, seed=3)
        want, want_lse, tol, lse_tol = ref.attention(con.Joined(own, shared, [0, 0, 1]), q, True, None)
        (k, v, ptable, pl, table, sl), scales = on(device, own, shared)
        if not any(lens):
            table = table[:, :0]
        if not any(plens):
            ptable = ptable[:, :0]
        cu = torch.tensor([0, 2, 3], dtype=torch.int32, device=device)
        o, lse = fa.flash_attention_paged_prefix(q.to(device), k, v, ptable, pl, table, sl, cu_prefix=cu,
                                                 return_lse=True, **scales)
        ref.check(o, want, tol * (1 + 2.0 ** -4), "O")
        ref.check(lse, want_lse, lse_tol + 2.0 ** -15, "LSE")


def test_prefix_more_new_tokens_than_keys(device):
    """Tokens that see no own key see their prefix; without one they get zeros and LSE -inf."""
    own, shared = Cache([3, 0, 40, 0], 2, 64, 16, BF16, False, news=[5, 2, 41, 2]), Cache([50], 2, 64, 16, BF16, False, seed=3)
    o, lse = attend(own, shared, [0, 3], device, 4)
    assert (o[48:] == 0).all() and (lse[:, 48:] == -math.inf).all()


@pytest.mark.parametrize("q8", [False, True])
def test_prefix_missing_pages(device, q8):
    """Entries that name no page hide their keys, of the prefix and of the sequence."""
    own = Cache([100, 40, 33], 2, 64, 16, FP16, q8, news=[3, 2, 1], gone=[(0, 1), (2, 0), (2, 1), (2, 2)])
    shared = Cache([200, 48], 2, 64, 16, FP16, q8, seed=3, gone=[(0, 0), (0, 5), (1, 0), (1, 1), (1, 2)])
    for i, x in ((3, 2 ** 31 - 1), (4, -2 ** 31), (6, 10 ** 6)):
        shared.table[0, i] = x
    o, lse = attend(own, shared, [0, 2, 3], device, 4)
    assert (o[5] == 0).all() and (lse[:, 5] == -math.inf).all()


def test_prefix_length_past_the_table(device):
    own, shared = Cache([20, 30], 2, 64, 16, FP16, False), Cache([100], 2, 64, 16, FP16, False, seed=3, width=4)
    attend(own, shared, None, device, 4)


@pytest.mark.parametrize("q8", [False, True])
def test_prefix_strided(device, q8):
    """[pages, page, H, D] storage, Q a slice of a wider projection, O written in place beside other rows."""
    own, shared = Cache([50, 129], 2, 64, 32, FP16, q8, news=[5, 20]), Cache([77], 2, 64, 32, FP16, q8, seed=3)
    attend(own, shared, None, device, 4, strided=True)
    args, kw = on(device, own, shared, True)
    wide = torch.randn(28, 12, 64, generator=torch.Generator().manual_seed(3)).half().to(device)
    out = torch.full((28, 6, 64), 5.0, dtype=FP16, device=device)
    got = fa.flash_attention_paged_prefix(wide[:, 2:6], *args, cu_seqlens=own.cu.to(device), out=out[:, 1:5], **kw)
    assert got.data_ptr() == out[:, 1:5].data_ptr()
    want, _, tol, _ = ref.attention(con.Joined(own, shared, [0, 0]), wide[:25, 2:6].cpu())
    ref.check(out[:25, 1:5], want, tol * (1 + 2.0 ** -4), "O")
    assert (out[:, 0] == 5).all() and (out[:, 5] == 5).all() and (out[25:] == 5).all()  # rows behind the last


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-9, 2.0])
def test_prefix_scales(device, scale):
    own, shared = Cache([20, 10], 2, 64, 16, BF16, False, news=[2, 1]), Cache([200], 2, 64, 16, BF16, False, seed=3)
    attend(own, shared, None, device, 4, scale=scale)


@pytest.mark.parametrize("first", [True, False])
def test_prefix_peaked(device, first):
    """All the weight on the prefix, or all of it on the own keys: the other state joins with weight 0."""
    own, shared = Cache([30, 9], 1, 64, 16, FP16, False, news=[3, 1]), Cache([90], 1, 64, 16, FP16, False, seed=3)
    for c, up in ((shared, first), (own, not first)):
        for b, n in enumerate(c.lens):
            k = c.rows[b][0] * 0.1 + (30.0 if up else -30.0)
            for j in range(n):
                c.k[int(c.table[b, j // 16]), :, j % 16] = k[:, j].half()
            c.rows[b][0] = k.half().double()
    attend(own, shared, None, device, 4)


def test_prefix_nonfinite(device):
    """A prefix row that is NaN reaches its group's sequences only; a NaN query its own row only."""
    own, shared = Cache([20, 30, 40], 1, 64, 16, BF16, False), Cache([64, 70], 1, 64, 16, BF16, False, seed=3)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    joined = con.Joined(own, shared, [0, 1, None])
    want, _, tol, _ = ref.attention(joined, q)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    q[2, 1] = math.nan
    shared.k[int(shared.table[0, 2]), 0, 5] = math.nan
    args, _ = on(device, own, shared)
    o, lse = fa.flash_attention_paged_prefix(q.to(device), *args, cu_prefix=cu, return_lse=True)
    assert o[0].isnan().all() and o[2, 1].isnan().all() and lse[1, 2].isnan() and lse[:, 0].isnan().all()
    ref.check(o[1], want[1], tol[1] * (1 + 2.0 ** -4), "O")
    for h in (0, 2, 3):
        ref.check(o[2, h], want[2, h], tol[2, h] * (1 + 2.0 ** -4), "O")


@pytest.mark.parametrize("news", [[1, 1, 1], [5, 3, 8], [70, 5, 33]])
@pytest.mark.parametrize("which", ["prefix", "own", "all of a prefix"])
def test_prefix_infinite_keys(device, news, which):
    """Keys that all rows score -inf have no part in O and LSE, alone in a tile or a whole prefix of them."""
    lens = [max(n, x) for n, x in zip(news, [20, 90, 40])]
    own, shared = Cache(lens, 1, 64, 16, BF16, False, news=news), Cache([64, 70], 1, 64, 16, BF16, False, seed=3)
    at = {"prefix": [(shared, 0, 3), (shared, 0, 33), (shared, 1, 69)], "own": [(own, 0, 2), (own, 1, 40)],
          "all of a prefix": [(shared, 1, j) for j in range(70)]}[which]
    q = torch.rand(sum(news), 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16() + 0.125
    joined = con.Joined(own, shared, [0, 1, None])  # of it those keys are left out
    left = [joined.held(b) for b in range(3)]
    for c, b, j in at:
        c.k[int(c.table[b, j // 16]), 0, j % 16, 7] = -math.inf
        c.rows[b][0][0, j, 7] = -math.inf
        left[b][j + (len(left[b]) - own.lens[b] if c is own else 0)] = False
    joined.held = lambda b: left[b]
    want, want_lse, tol, lse_tol = ref.attention(joined, q)
    tol, lse_tol = tol * (1 + 2.0 ** -4), lse_tol + 2.0 ** -15  # (as in attend)
    args, _ = on(device, own, shared)
    pools, table, rest = args[:2], args[2], args[3:]
    wide = torch.nn.functional.pad(table, (0, (160 << 20) // (3 * 256 * 16)), value=-1)
    for t in (table, wide):
        for hint in (1, 10 ** 6):
            o, lse = fa.flash_attention_paged_prefix(
                q.to(device), *pools, t, *rest, cu_seqlens=own.cu.to(device), max_query_len=hint, return_lse=True,
                cu_prefix=torch.tensor([0, 1, 2], dtype=torch.int32, device=device))
            ref.check(o, want, tol, f"O (hint {hint})")
            ref.check(lse, want_lse, lse_tol, f"LSE (hint {hint})")


def test_prefix_indexes_are_held_to_their_ranges(device):
    """cu_prefix and cu_seqlens that fall or pass their ends: nothing outside the rows is written."""
    own, shared = Cache([50, 30], 2, 64, 16, FP16, False, news=[3, 1]), Cache([50, 20], 2, 64, 16, FP16, False, seed=3)
    args, q = on(device, own, shared)[0], torch.randn(4, 4, 64).half().to(device)
    big = 2 ** 31 - 1
    for cu in ([0, 3, 4], [0, -5, 4], [big, 0, 1], [-2 ** 31, 2, big], [4, 4, 4]):
        for cup in ([0, 1, 2], [-7, 100, 3], [big, -big, big], [2, 1, 0], [0, 2, 1]):
            room = torch.full((12, 4, 64), 7.0, dtype=FP16, device=device)
            fa.flash_attention_paged_prefix(q, *args, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device),
                                            cu_prefix=torch.tensor(cup, dtype=torch.int32, device=device), out=room[4:8])
            assert (room[:4] == 7).all() and (room[8:] == 7).all()
    lens = torch.tensor([-5, -2 ** 31], dtype=torch.int32, device=device)
    o = fa.flash_attention_paged_prefix(q[:2], *args[:3], lens, args[4], lens,
                                        cu_prefix=torch.tensor([0, 1, 2], dtype=torch.int32, device=device))
    assert (o == 0).all()


def test_prefix_nothing_to_do(device):
    own, shared = Cache([5], 2, 64, 16, FP16, False), Cache([20], 2, 64, 16, FP16, False, seed=3)
    k, v, ptable, plens, table, lens = on(device, own, shared)[0]
    empty, cu = torch.empty(0, 4, 64, dtype=FP16, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    assert fa.flash_attention_paged_prefix(empty, k, v, ptable, plens, table, lens, cu_seqlens=cu).shape == (0, 4, 64)
    q = torch.randn(1, 4, 64).half().to(device)
    none = fa.flash_attention_paged_prefix(q, k, v, ptable[:0], plens[:0], table, lens, cu_prefix=cu[:1])  # no prefix
    assert torch.equal(none, fa.flash_attention_paged(q, k, v, table, lens))
    o, lse = fa.flash_attention_paged_prefix(q, k[:0], v[:0], ptable, plens, table, lens, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()  # a pool without pages
    wide = fa.flash_attention_paged_prefix(q, k, v, ptable[:, :0], plens, table, lens)  # a prefix table without columns
    ref.check(wide, none.cpu().double(), 2 * ref.U[FP16] * none.cpu().double().abs() + 2.0 ** -24, "O")


def test_prefix_same_bits_every_time(device):
    own, shared = Cache([300, 17, 90] * 9, 2, 128, 16, BF16, True), Cache([3000], 2, 128, 16, BF16, True, seed=3)
    first = attend(own, shared, None, device, 8)
    for _ in range(3):
        again = attend(own, shared, None, device, 8)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_prefix_out_that_overlaps_is_refused(device):
    own, shared = Cache([50], 2, 64, 32, FP16, False), Cache([50], 2, 64, 32, FP16, False, seed=3)
    args = on(device, own, shared)[0]
    q = torch.zeros(1, 4, 64, dtype=FP16, device=device)
    for out in (q, args[0].view(-1, 4, 64)[:1]):
        with pytest.raises(RuntimeError, match="must not share"):
            fa.flash_attention_paged_prefix(q, *args, out=out)


# ---- weights ------------------------------------------------------------------------------


def lse_of(c, q, device, causal=True, scale=None):
    (args, kw) = c.args(device)
    return fa.flash_attention_paged(q.to(device), *args, cu_seqlens=c.cu.to(device), scale=scale,
                                    causal="bottom_right" if causal else False, return_lse=True, **kw)[1]


def weigh(c, device, hq, seed=1, causal=True, scale=None, strided=False, max_len=None):
    """The call with each hint, new and added to what is there, checked; returns the weights."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(c.news), hq, c.d, generator=g).to(c.dtype)
    lse = lse_of(c, q, device, causal, scale)
    want, tol = con.weights(c, q, lse.cpu(), causal, scale, max_len)
    (args, kw) = c.args(device, strided)
    kw = {"k_scale": kw["k_scale"]} if kw else {}
    ones = all(n == 1 for n in c.news)
    kw.update(causal="bottom_right" if causal else False, scale=scale, cu_seqlens=None if ones else c.cu.to(device))
    held = torch.zeros(want.shape[0], want.shape[2], dtype=torch.bool)
    for b in range(len(c.lens)):
        x = c.held(b)[:want.shape[2]]
        held[b, :len(x)] = x
    for hint in [None] if ones else [1, 10 ** 6]:
        w = fa.paged_attention_weights(q.to(device), lse, args[0], *args[2:], max_len=max_len, max_query_len=hint, **kw)
        ref.check(w, want, tol, f"weights (max_query_len={hint})")
        # Into a slice of a wider tensor: the sum rounds once.
        wide = torch.rand(want.shape[0], c.hkv + 1, want.shape[2] + 3, generator=g).to(device)
        before = wide.clone()
        to = wide[:, 1:, 2:2 + want.shape[2]]
        got = fa.paged_attention_weights(q.to(device), lse, args[0], *args[2:], max_query_len=hint, add_to=to, **kw)
        assert got.data_ptr() == to.data_ptr()
        base = before[:, 1:, 2:2 + want.shape[2]].cpu().double()
        ref.check(got, want + base, tol + 2.0 ** -24 * (want + base + tol), "added weights")
        to.copy_(before[:, 1:, 2:2 + want.shape[2]].clone())
        assert torch.equal(wide, before)  # nothing beside them
        assert torch.equal(got.cpu()[:, :, :][~held[:, None].expand_as(want)], base.float()[~held[:, None].expand_as(want)])
    return w


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_weights_single_tokens(device, d, dtype, q8, page):
    c = Cache([1, 0, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 300, 1000], 2, d, page, dtype, q8)
    w = weigh(c, device, 8)
    live = torch.tensor([n > 0 for n in c.lens])
    assert (w.cpu().sum(-1)[live] - 4).abs().max() < 1e-3  # of 4 query heads each


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (14, 2), (12, 12), (32, 8), (15, 3), (40, 2), (16, 16)])
@pytest.mark.parametrize("q8", [False, True])
def test_weights_heads(device, hq, hkv, q8):
    weigh(Cache([77, 300, 5], hkv, 64, 16, BF16, q8), device, hq)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news", [[4, 4, 4], [1, 9, 2], [0, 3, 0], [70, 5, 33], [130, 1, 257]])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_chunks(device, d, q8, news, causal):
    lens = [max(n, x) for n, x in zip(news, [130, 200, 257])]
    weigh(Cache(lens, 2, d, 16, FP16, q8, news=news), device, 6, causal=causal)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_weights_long(device, d, q8):
    weigh(Cache([5000, 3, 2500, 64], 2, d, 32, BF16, q8), device, 8)
    weigh(Cache([2500, 3, 700, 64], 2, d, 16, BF16, q8, news=[40, 2, 1, 64]), device, 8)
    weigh(Cache([900], 1, d, 16, FP16, q8, news=[900]), device, 4)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 1), (7, 1), (14, 2), (100, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_prompts(device, hq, hkv, causal):
    """Blocks of new keys, which fewer rows see, next to old ones, dealt in equal stretches."""
    weigh(Cache([1500], hkv, 64, 16, FP16, False, news=[1500]), device, hq, causal=causal)
    weigh(Cache([1000, 0, 700, 300], hkv, 128, 16, BF16, True, news=[333, 0, 1000, 7]), device, hq, causal=causal)


def test_weights_prompts_of_many_sequences(device):
    lens = [(37 * i) % 301 for i in range(70)]
    weigh(Cache(lens, 2, 64, 16, BF16, False, news=[max(0, x - (i % 3) * 50) for i, x in enumerate(lens)]), device, 6)


@pytest.mark.parametrize("max_len", [1, 256, 700, 1700])
def test_weights_prompts_max_len(device, max_len):
    w = weigh(Cache([1500, 90], 2, 64, 16, FP16, False, news=[1100, 80]), device, 8, max_len=max_len)
    assert w.shape == (2, 2, max_len)


@pytest.mark.parametrize("max_len", [1, 31, 33, 100, 333, 1000])
def test_weights_max_len(device, max_len):
    """Positions past max_len are not weighed, those past the sequence get 0; rows still see all keys."""
    c = Cache([300, 64, 5], 2, 64, 16, FP16, False, news=[3, 1, 5])
    w = weigh(c, device, 4, max_len=max_len)
    assert w.shape == (3, 2, max_len) and (w[1:, :, 64:] == 0).all()


def test_weights_more_new_tokens_than_keys(device):
    w = weigh(Cache([3, 0, 40], 2, 64, 16, BF16, False, news=[5, 2, 41]), device, 4)
    assert (w[1] == 0).all() and abs(float(w[0, 0].sum()) - 6) < 1e-3  # three of five tokens, two heads


@pytest.mark.parametrize("q8", [False, True])
def test_weights_missing_pages(device, q8):
    c = Cache([500, 100, 40, 33], 2, 64, 16, FP16, q8, news=[3, 1, 2, 70],
              gone=[(0, i) for i in range(9)] + [(1, 6), (2, 0), (2, 1), (2, 2)])
    for i, x in zip((3, 4, 5, 6), [c.k.shape[0], 2 ** 31 - 1, -2 ** 31, -7]):
        c.table[0, i] = x
    weigh(c, device, 4)


def test_weights_shared_pages(device):
    c = Cache([96, 96, 50], 2, 64, 16, BF16, True)
    c.table[1, :4] = c.table[0, :4]
    c.table[1, 5] = c.table[1, 4]  # and a page twice in one sequence
    for x in range(2):
        c.rows[1][x][:, :64] = c.rows[0][x][:, :64]
        c.rows[1][x][:, 80:] = c.rows[1][x][:, 64:80]
    weigh(c, device, 6)


@pytest.mark.parametrize("q8", [False, True])
def test_weights_strided(device, q8):
    weigh(Cache([50, 129], 2, 64, 32, FP16, q8, news=[5, 20]), device, 4, strided=True)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-9, 1.0])
def test_weights_scales(device, scale):
    weigh(Cache([200, 10], 2, 64, 16, BF16, False, news=[2, 1]), device, 4, scale=scale)


@pytest.mark.parametrize("news", [[1, 1], [40, 3]])
def test_weights_nonfinite(device, news):
    """Rows of LSE -inf add nothing; a NaN key gives its own weight only; a NaN LSE those its row sees."""
    c = Cache([400, 90], 1, 64, 16, BF16, False, news=news)
    q = torch.randn(sum(news), 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    lse = lse_of(c, q, device)
    lse[1, 0] = -math.inf
    want, tol = con.weights(c, q, lse.cpu())
    p = int(c.table[0, 5])
    c.k[p, 0, 3] = math.nan
    (args, _) = c.args(device)
    for hint in (1, 10 ** 6):
        w = fa.paged_attention_weights(q.to(device), lse, args[0], *args[2:], cu_seqlens=c.cu.to(device), max_query_len=hint)
        assert w[0, 0, 83].isnan() and int(w.isnan().sum()) == 1
        keep = torch.ones_like(want, dtype=torch.bool)
        keep[0, 0, 83] = False
        ref.check(w.cpu()[keep], want[keep], tol[keep], "weights")
        bad = lse.clone()
        bad[2, -1] = math.nan
        w = fa.paged_attention_weights(q.to(device), bad, args[0], *args[2:], cu_seqlens=c.cu.to(device), max_query_len=hint)
        assert w[1, 0, :90].isnan().all() and (w[1, 0, 90:] == 0).all() and int(w[0].isnan().sum()) == 1


@pytest.mark.parametrize("news", [[1, 1], [5, 3], [40, 3], [130, 90]])
@pytest.mark.parametrize("at", [0, 3, 60, 255, 395, 399])
@pytest.mark.parametrize("scale", [None, -0.3])
def test_weights_infinite_key(device, news, at, scale):
    """A key that all rows score -inf has weight 0, wherever it stands and whatever the number of rows."""
    c = Cache([400, 90], 1, 64, 16, BF16, False, news=news)
    q = torch.rand(sum(news), 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16() + 0.125
    c.k[int(c.table[0, at // 16]), 0, at % 16, 7] = -math.inf if scale is None else math.inf
    c.rows[0][0][0, at, 7] = -math.inf if scale is None else math.inf
    lse = lse_of(c, q, device, scale=scale)
    assert lse.isfinite().all()  # attention gives the key no weight
    want, tol = con.weights(c, q, lse.cpu(), scale=scale)
    assert want[0, 0, at] == 0 and not want.isnan().any()
    (args, _) = c.args(device)
    for hint in (1, 10 ** 6):
        w = fa.paged_attention_weights(q.to(device), lse, args[0], *args[2:], cu_seqlens=c.cu.to(device), scale=scale,
                                       max_query_len=hint)
        ref.check(w, want, tol, f"weights (hint {hint})")
        assert w[0, 0, at] == 0


@pytest.mark.parametrize("news", [[1, 1], [5, 3], [40, 3], [130, 90]])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_rows_left_out(device, news, causal):
    """A row of LSE -inf adds nothing, whatever its query and the keys hold: the last row, the first, all of a sequence's.
    One of LSE +inf gives finite scores 0."""
    c = Cache([400, 90], 1, 64, 16, BF16, False, news=news)
    q = torch.randn(sum(news), 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    lse = lse_of(c, q, device, causal)
    out = [(0, 0), (3, news[0] - 1)] + [(h, t) for h in range(4) for t in range(news[0], sum(news))]
    for h, t in out:
        lse[h, t] = -math.inf
        q[t, h, 5] = math.nan
    lse[1, 0] = math.inf
    # What only rows that are left out see: the last sequence's keys.
    for j, x in ((2, math.inf), (33, math.nan), (70, -math.inf)):
        c.k[int(c.table[1, j // 16]), 0, j % 16, 7] = x
    rows = q.clone()
    for h, t in out:
        rows[t, h] = 0
    want, tol = con.weights(c, rows, lse.cpu(), causal)
    assert (want[1] == 0).all() and want.isfinite().all()
    (args, _) = c.args(device)
    for hint in (1, 10 ** 6):
        w = fa.paged_attention_weights(q.to(device), lse, args[0], *args[2:], cu_seqlens=c.cu.to(device), max_query_len=hint,
                                       causal="bottom_right" if causal else False)
        ref.check(w, want, tol, f"weights (hint {hint})")
        assert (w[1] == 0).all()


def test_weights_indexes_are_held_to_their_ranges(device):
    c = Cache([50, 30], 2, 64, 16, FP16, False, news=[3, 1])
    (args, _), q = c.args(device), torch.randn(4, 4, 64).half().to(device)
    lse = torch.zeros(4, 4, device=device)
    for cu in ([0, 3, 100], [0, -5, 4], [2 ** 31 - 1, 0, 1], [-2 ** 31, 2, 2 ** 31 - 1], [4, 4, 4]):
        room = torch.full((6, 2, 64), 7.0, device=device)
        for hint in (1, 10 ** 6):
            fa.paged_attention_weights(q, lse, args[0], *args[2:], add_to=room[2:4], max_query_len=hint,
                                       cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=device))
        assert (room[:2] == 7).all() and (room[4:] == 7).all()
    lens = torch.tensor([-5, 2 ** 31 - 1], dtype=torch.int32, device=device)
    w = fa.paged_attention_weights(q, lse, args[0], args[2], lens, cu_seqlens=c.cu.to(device), causal=False)
    assert (w[0] == 0).all()


def test_weights_nothing_to_do(device):
    c = Cache([5, 20], 2, 64, 16, FP16, False)
    (k, v, table, lens), _ = c.args(device)
    empty, cu = torch.empty(0, 4, 64, dtype=FP16, device=device), torch.zeros(3, dtype=torch.int32, device=device)
    none = torch.empty(4, 0, device=device)
    w = fa.paged_attention_weights(empty, none, k, table, lens, cu_seqlens=cu)  # no new token: no weight
    assert w.shape == (2, 2, 32) and (w == 0).all()
    to = torch.full((2, 2, 32), 3.0, device=device)
    fa.paged_attention_weights(empty, none, k, table, lens, cu_seqlens=cu, add_to=to)
    assert (to == 3).all()
    assert fa.paged_attention_weights(empty, none, k, table[:0], lens[:0]).shape == (0, 2, 32)
    q, lse = torch.randn(2, 4, 64).half().to(device), torch.zeros(4, 2, device=device)
    assert fa.paged_attention_weights(q, lse, k, table, lens, max_len=0).shape == (2, 2, 0)
    assert (fa.paged_attention_weights(q, lse, k[:0], table, lens) == 0).all()
    assert fa.paged_attention_weights(q, lse, k, table[:, :0], lens).shape == (2, 2, 0)
    assert (fa.paged_attention_weights(q, lse, k, table[:, :0], lens, max_len=40) == 0).all()


def test_weights_refusals(device):
    c = Cache([50, 30], 2, 64, 16, FP16, False)
    (k, v, table, lens), _ = c.args(device)
    q, lse = torch.randn(2, 4, 64).half().to(device), torch.zeros(4, 2, device=device)
    to = torch.zeros(2, 2, 64, device=device)
    call = lambda lse=lse, to=to, q=q, **kw: fa.paged_attention_weights(q, lse, k, table, lens, add_to=to, **kw)  # noqa: E731
    for bad, msg in ((dict(lse=lse.double()), "LSE must be float32"), (dict(lse=lse[:3]), r"\[H_q, tokens\]"),
                     (dict(lse=lse.cpu()), "cache's device"), (dict(to=to.half()), "add_to must be float32"),
                     (dict(to=to[:1]), r"\[B, H_kv, max_len\]"), (dict(to=to.cpu()), "cache's device"),
                     (dict(to=to.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
                     (dict(to=to[:1].expand(2, 2, 64)), "overlap"),
                     (dict(to=torch.zeros(300, device=device).as_strided((2, 2, 64), (100, 50, 1))), "overlap"),
                     (dict(q=q.to(BF16)), "cache's dtype"), (dict(scale=math.inf), "finite")):
        with pytest.raises(RuntimeError, match=msg):
            call(**bad)
    over = k.view(-1).view(torch.float32)[:256].view(2, 2, 64)
    with pytest.raises(RuntimeError, match="must not share"):
        call(to=over)
    with pytest.raises(ValueError, match="max_len"):
        call(max_len=10)


# ---- eviction ---------------------------------------------------------------------------


def evict(c, device, keep, recent, seed=1, extra=1, w=None, strided=False, wide=False):
    """The call on a cache whose pool has `extra` more pages for each sequence than needed, checked."""
    g = torch.Generator().manual_seed(seed)
    room = c.width * c.page
    if w is None:
        w = torch.exp(2 * torch.randn(len(c.lens), c.hkv, room, generator=g))
    need = -(-min(keep, room) // c.page) + extra
    pools = [c.k, c.v] + ([c.ks, c.vs] if c.q8 else [])
    more = []
    for x in pools:
        y = (torch.rand(len(c.lens) * need, *x.shape[1:], generator=g) * 100).to(torch.uint8)
        more.append(torch.cat([x.view(torch.uint8), y]).view(x.dtype) if x.element_size() == 1
                    else torch.cat([x, y.to(x.dtype)]))
    order = torch.randperm(len(c.lens) * need, generator=g) + c.pages
    to = order.view(len(c.lens), need).int()
    want = con.evicted(c, more, w, to, keep, recent)
    back = c.k, c.v, c.ks, c.vs
    c.k, c.v, *scales = more
    if scales:
        c.ks, c.vs = scales
    (args, kw) = c.args(device, strided)
    c.k, c.v, c.ks, c.vs = back
    wd = w.to(device)
    if wide:  # a slice of a wider tensor, longer than the tables
        wd = torch.full((len(c.lens), c.hkv + 1, room + 7), 9e9, device=device)[:, 1:]
        wd[:, :, :room] = w.to(device)
    lens, left = fa.paged_cache_evict(*args, wd, to.to(device), keep, recent, **kw)
    assert torch.equal(lens.cpu(), want[1])
    assert torch.equal(left.cpu().view(torch.int32), want[2].view(torch.int32))
    got = [args[0], args[1]] + ([kw["k_scale"], kw["v_scale"]] if c.q8 else [])
    for x, y in zip(got, want[0]):
        bits = torch.uint8 if x.element_size() == 1 else torch.int16
        assert torch.equal(x.cpu().contiguous().view(bits), y.view(bits))
    assert torch.equal(args[2].cpu(), c.table) and torch.equal(args[3].cpu(), c.seq_lens)
    return args, kw, lens, left, to


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (16, 3), (100, 100), (129, 0), (333, 64)])
def test_evict(device, d, q8, page, keep, recent):
    evict(Cache([1, 0, 15, 16, 17, 64, 127, 128, 129, 130, 500], 2, d, page, FP16, q8), device, keep, recent)


@pytest.mark.parametrize("hkv", [1, 3, 12])
def test_evict_heads(device, hkv):
    evict(Cache([300, 77, 1025], hkv, 64, 16, BF16, False), device, 200, 20, wide=True)


@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 1), (33000, 5), (20000, 1000), (40000, 0)])
def test_evict_long(device, keep, recent):
    """Rows of several workgroups, one of few positions among them."""
    evict(Cache([34567, 100, 8192, 8193, 0], 1, 64, 128, BF16, True), device, keep, recent)


@pytest.mark.parametrize("keep,recent", [(4000, 100), (16000, 0)])
def test_evict_blocks(device, keep, recent):
    """Sizes at a block's borders, ties over several of them, pages missing in some."""
    c = Cache([16384, 16383, 16385, 9000], 2, 64, 256, FP16, False, gone=[(3, 0), (0, 31), (0, 32), (0, 33), (2, 63)])
    w = torch.randint(0, 6, (4, 2, c.width * 256), generator=torch.Generator().manual_seed(6)).float()
    evict(c, device, keep, recent, w=w)


def test_evict_many_blocks_of_a_workgroup(device):
    """More rows than workgroups are wanted: each takes several blocks."""
    batch, room, keep = 2100, 16384 + 256, 5
    g = torch.Generator().manual_seed(3)
    k = torch.randn(3 + batch, 2, 256, 64, generator=g).half().to(device)
    table = torch.zeros(batch, room // 256, dtype=torch.int32, device=device)
    table[:, 1::2] = 1
    lens = torch.randint(room - 300, room + 1, (batch,), generator=g).int().to(device)
    to = torch.arange(3, 3 + batch, dtype=torch.int32, device=device)[:, None]
    w = torch.rand(batch, 2, room, generator=g).to(device)
    old = k.clone()
    got, left = fa.paged_cache_evict(k, k.clone(), table, lens, w, to, keep)
    assert (got == keep).all()
    live = torch.where(torch.arange(room, device=device) < lens[:, None, None], w, -1.0)
    at = live.topk(keep).indices.sort(-1).values
    assert torch.equal(left[:, :, :keep], w.gather(2, at)) and (left[:, :, keep:] == 0).all()
    want = old[(at // 256) % 2, torch.arange(2, device=device)[:, None], at % 256]
    assert torch.equal(k[3:, :, :keep], want)


@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 1), (700, 33), (9000, 0), (17000, 0)])
def test_evict_many_long_rows(device, keep, recent):
    """Rows of several blocks, of each a workgroup: lengths at a block's borders and none, ties, pages missing."""
    lens = [17000, 8191, 8192, 8193, 0, 1, 16384, 16385, 9999] + [(61 * i) % 400 for i in range(57)]
    c = Cache(lens, 2, 64, 256, BF16, False, gone=[(0, 0), (0, 32), (3, 32), (6, 5)])
    g = torch.Generator().manual_seed(6)
    w = torch.rand(66, 2, c.width * 256, generator=g)
    w[:9] = torch.randint(0, 6, w[:9].shape, generator=g).float()
    w[7, 1, ::3] = math.nan
    evict(c, device, keep, recent, w=w)


@pytest.mark.parametrize("q8", [False, True])
def test_evict_missing_pages(device, q8):
    """Positions without a page hold no row: what stays closes up; to_table may lack pages too."""
    c = Cache([500, 100, 40, 33], 2, 64, 16, FP16, q8,
              gone=[(0, i) for i in range(9)] + [(0, 20), (1, 6), (2, 0), (2, 1), (2, 2)])
    for i, x in zip((3, 4, 5, 6), [c.k.shape[0] + 1000, 2 ** 31 - 1, -2 ** 31, -7]):
        c.table[0, i] = x
    for keep, recent in ((50, 10), (100, 100), (400, 0)):
        evict(c, device, keep, recent)


def test_evict_to_missing_pages(device):
    """Rows whose place has no page are dropped, the others and all weights arrive."""
    c = Cache([200, 90], 2, 64, 16, FP16, False)
    w = torch.rand(2, 2, c.width * 16, generator=torch.Generator().manual_seed(1))
    pool = torch.cat([c.k, torch.zeros(8, *c.k.shape[1:], dtype=FP16)])
    to = torch.arange(c.pages, c.pages + 8).view(2, 4).int()
    to[0, 1], to[1, 2] = -1, 2 ** 31 - 1
    want = con.evicted(c, [pool, pool], w, to, 60, 5)
    k, v = pool.clone().to(device), pool.clone().to(device)
    lens, left = fa.paged_cache_evict(k, v, c.table.to(device), c.seq_lens.to(device), w.to(device), to.to(device), 60, 5)
    assert lens.tolist() == [60, 60] and torch.equal(left.cpu(), want[2])
    assert torch.equal(k.cpu().view(torch.int16), want[0][0].view(torch.int16))
    assert torch.equal(v.cpu().view(torch.int16), want[0][1].view(torch.int16))


def test_evict_ties_and_special_weights(device):
    """Equal weights go to the lowest positions; zeros of both signs are equal, NaN is least, infinities count."""
    c = Cache([200, 200, 200, 200], 2, 64, 16, FP16, False)
    g = torch.Generator().manual_seed(4)
    w = torch.zeros(4, 2, c.width * 16)
    w[0] = torch.randint(0, 3, w[0].shape, generator=g).float()
    w[1] = torch.where(torch.rand(w[1].shape, generator=g) < 0.5, -0.0, 0.0)
    w[2] = torch.randint(-2, 3, w[2].shape, generator=g).float()
    w[2][torch.rand(w[2].shape, generator=g) < 0.5] = math.nan
    w[3] = torch.randn(w[3].shape, generator=g)
    w[3, :, ::7], w[3, :, ::5], w[3, :, ::11] = math.inf, -math.inf, math.nan
    w[3, 1, 3::4] = 1e-42
    for keep, recent in ((7, 0), (64, 9), (120, 0), (199, 0), (150, 150)):
        evict(c, device, keep, recent, w=w)


@pytest.mark.parametrize("q8", [False, True])
def test_evict_strided(device, q8):
    evict(Cache([500, 77], 3, 64, 16, BF16, q8), device, 100, 30, strided=True, wide=True)


def test_evict_shared_pages(device):
    """Sequences that share pages each get their own rows of them."""
    c = Cache([96, 96, 50], 2, 64, 16, BF16, True)
    c.table[1, :4] = c.table[0, :4]
    evict(c, device, 40, 8)


def test_evict_length_past_the_table(device):
    """seq_lens past the table's room: the recent positions lie behind it, and what it holds competes."""
    c = Cache([100, 90], 2, 64, 16, FP16, False, width=3)
    evict(c, device, 20, 10)
    evict(c, device, 64, 64)


def test_evict_many_sequences(device):
    evict(Cache([(37 * i) % 90 for i in range(150)], 2, 64, 16, FP16, True), device, 33, 4)


def test_evict_indexes_are_held_to_their_ranges(device):
    c = Cache([50, 30], 2, 64, 16, FP16, False)
    (args, _) = c.args(device)
    w, to = torch.rand(2, 2, 64, device=device), torch.tensor([[-1], [2 ** 31 - 1]], dtype=torch.int32, device=device)
    before = args[0].clone()
    for lens in ([-5, -2 ** 31], [2 ** 31 - 1, 10 ** 9]):
        got, left = fa.paged_cache_evict(*args[:3], torch.tensor(lens, dtype=torch.int32, device=device), w, to, 9, 9)
        assert torch.equal(args[0].view(torch.int16), before.view(torch.int16))
        assert (left[:, :, 9:] == 0).all() and got.tolist() == ([0, 0] if lens[0] < 0 else [9, 9])


def test_evict_nothing_to_do(device):
    c = Cache([5, 20], 2, 64, 16, FP16, False)
    (k, v, table, lens), _ = c.args(device)
    w, to = torch.rand(2, 2, 32, device=device), torch.full((2, 2), -1, dtype=torch.int32, device=device)
    got, left = fa.paged_cache_evict(k, v, table[:0], lens[:0], w[:0], to[:0], 5)
    assert got.shape == (0,) and left.shape == (0, 2, 32)
    got, left = fa.paged_cache_evict(k, v, table, lens, w, to[:, :0], 0)
    assert got.tolist() == [0, 0] and left.shape == (2, 2, 0)
    got, left = fa.paged_cache_evict(k, v, table[:, :0], lens, w, to, 7)
    assert got.tolist() == [0, 0] and (left == 0).all()
    got, left = fa.paged_cache_evict(k[:0], v[:0], table, lens, w, to, 7)
    assert got.tolist() == [0, 0] and (left == 0).all()


def test_evict_refusals(device):
    c = Cache([50, 30], 2, 64, 16, FP16, False)
    (k, v, table, lens), _ = c.args(device)
    w, to = torch.rand(2, 2, 64, device=device), torch.zeros(2, 2, dtype=torch.int32, device=device)
    call = lambda w=w, to=to, keep=20, recent=0, k=k: fa.paged_cache_evict(k, v, table, lens, w, to, keep, recent)  # noqa: E731
    for bad, msg in ((dict(w=w[:, :, :63]), "block_table's room"), (dict(w=w.double()), "float32"),
                     (dict(w=w.cpu()), "cache's device"), (dict(w=w[:, :1]), r"\[B, H_kv, max_len\]"),
                     (dict(to=to.long()), "int32"), (dict(to=to[:1]), "same batch"), (dict(to=to[:, :1]), "room for 16 rows, up to 20"),
                     (dict(keep=33), "room for 32 rows, up to 33"), (dict(keep=10 ** 12), "room for 32 rows, up to 64"),
                     (dict(keep=-1), "non-negative"), (dict(recent=-1), "non-negative"),
                     (dict(recent=21), "must not exceed keep"), (dict(k=k[:1].expand_as(k)), "expanded")):
        with pytest.raises(RuntimeError, match=msg):
            call(**bad)


# ---- versions, streams, graphs ---------------------------------------------------------------


def test_what_is_written_counts_as_changed(device):
    c = Cache([50, 30], 2, 64, 16, FP16, True)
    (args, kw) = c.args(device)
    tensors = [args[0], args[1], *kw.values()]
    before = [t._version for t in tensors]
    w, to = torch.rand(2, 2, 64, device=device), torch.full((2, 2), -1, dtype=torch.int32, device=device)
    fa.paged_cache_evict(*args, w, to, 20, **kw)
    assert all(t._version > x for t, x in zip(tensors, before))
    q, lse = torch.randn(2, 4, 64).half().to(device), torch.zeros(4, 2, device=device)
    n = w._version
    fa.paged_attention_weights(q, lse, args[0], *args[2:], k_scale=kw["k_scale"], add_to=w)
    assert w._version > n


def serve(own, shared, q, args, kw, to, state, hint):
    """A step of a server: attention behind a prefix, the weights of own and prefix rows, eviction."""
    k, v, ptable, plens, table, lens = args
    ks = {"k_scale": kw["k_scale"]} if kw else {}
    cu = state["cu"]
    o, lse = fa.flash_attention_paged_prefix(q, *args, cu_seqlens=cu, max_query_len=hint, return_lse=True, **kw)
    w = fa.paged_attention_weights(q, lse, k, table, lens, cu_seqlens=cu, max_query_len=hint, **ks)
    fa.paged_attention_weights(q, lse, k, ptable, plens, cu_seqlens=state["every"], causal=False,
                               add_to=state["prefix"], **ks)
    new_lens, kept = fa.paged_cache_evict(k, v, table, lens, w, to, 24, 6, **kw)
    again = fa.flash_attention_paged_prefix(q, k, v, ptable, plens, to, new_lens, cu_seqlens=cu, causal=False, **kw)
    return o, lse, w, new_lens, kept, again


def setting(device, q8, news, seed=0):
    own = Cache([40, 90, 17], 2, 64, 16, BF16, q8, news=news, seed=seed)
    shared = Cache([100], 2, 64, 16, BF16, q8, seed=seed + 1)
    args, kw = on(device, own, shared)
    pages = args[0].shape[0]
    grow = lambda x: torch.cat([x.view(torch.uint8), torch.zeros_like(x.view(torch.uint8))[:6]]).view(x.dtype)  # noqa: E731
    args = (grow(args[0]) if q8 else torch.cat([args[0], args[0][:6] * 0]),
            grow(args[1]) if q8 else torch.cat([args[1], args[1][:6] * 0]), *args[2:])
    kw = {n: grow(x) for n, x in kw.items()}
    to = torch.arange(pages, pages + 6, dtype=torch.int32, device=device).view(3, 2)
    t = sum(news)
    q = torch.randn(t, 8, 64, generator=torch.Generator().manual_seed(seed + 2)).bfloat16()
    state = {"cu": own.cu.to(device), "every": torch.tensor([0, t], dtype=torch.int32, device=device),
             "prefix": torch.zeros(1, 2, shared.width * 16, device=device)}
    return own, shared, q, args, kw, to, state


@pytest.mark.parametrize("news", [[1, 1, 1], [3, 40, 9]])
@pytest.mark.parametrize("q8", [False, True])
def test_together(device, q8, news):
    """Attention behind a prefix, the weights of all rows, eviction by them, attention over what is left."""
    own, shared, q, args, kw, to, state = setting(device, q8, news)
    o, lse, w, new_lens, kept, again = serve(own, shared, q.to(device), args, kw, to, state, None)
    joined = con.Joined(own, shared, [0, 0, 0])
    want, want_lse, tol, lse_tol = ref.attention(joined, q)
    ref.check(o, want, tol * (1 + 2.0 ** -4), "O")
    ref.check(lse, want_lse, lse_tol + 2.0 ** -15, "LSE")
    want_w, w_tol = con.weights(own, q, lse.cpu())
    ref.check(w, want_w, w_tol, "weights")
    shared.news, shared.cu = [sum(news)], torch.tensor([0, sum(news)], dtype=torch.int32)
    want_p, p_tol = con.weights(shared, q, lse.cpu(), causal=False)
    ref.check(state["prefix"], want_p, p_tol, "the prefix's weights")
    # Each row's probabilities, over its prefix and its own keys, add up to 1.
    total = float(w.double().sum() + state["prefix"].double().sum())
    assert abs(total - 8 * sum(news)) < 1e-3 * 8 * sum(news)
    left = [[con.stays(w[b, h].tolist(), own.held(b).tolist(), own.lens[b], 24, 6) for h in range(2)] for b in range(3)]
    assert new_lens.tolist() == [24, 24, 17]
    for b in range(3):
        for h in range(2):
            assert torch.equal(kept[b, h, :len(left[b][h])], w[b, h, left[b][h]])
            for x in range(2):
                joined.rows[b][x] = joined.rows[b][x].clone()
        for x in range(2):
            rows = torch.stack([own.rows[b][x][h, left[b][h]] for h in range(2)])
            joined.rows[b][x] = torch.cat([shared.rows[0][x], rows], 1)
        joined.lens[b] = 100 + len(left[b][0])
    joined.held = lambda b: torch.ones(joined.lens[b], dtype=torch.bool)
    want, _, tol, _ = ref.attention(joined, q, causal=False)
    ref.check(again, want, tol * (1 + 2.0 ** -4), "O over what is left")


def test_other_stream(device):
    """On a stream of their own, behind work that fills the inputs there."""
    own, shared, q, args, kw, to, state = setting(device, False, [3, 40, 9])
    first = serve(own, shared, q.to(device), args, kw, to, state, None)
    prefix = state["prefix"].clone()
    own, shared, q, args, kw, to, state = setting(device, False, [3, 40, 9])
    late, q = torch.empty_like(q, device=device), q.to(device)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        junk = torch.randn(4096, 4096, device=device)
        for _ in range(4):
            junk = junk @ junk * 1e-3
        late.copy_(q)
        got = serve(own, shared, late, args, kw, to, state, None)
    side.synchronize()
    for x, y in zip(first, got):
        assert torch.equal(x, y)
    assert torch.equal(prefix, state["prefix"])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("news", [[1, 1, 1], [3, 40, 9]])
def test_graph(device, q8, news):
    """Captured once, replayed on changed tables, lengths and queries, with eager work between; a second graph
    of the same calls replayed in turn."""
    own, shared, q, args, kw, to, state = setting(device, q8, news)
    q = q.to(device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        serve(own, shared, q, args, kw, to, state, None)
    side.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = serve(own, shared, q, args, kw, to, state, None)
        graphs.append((graph, outs))
    for i in range(6):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(50 + i)).bfloat16())
        args[5].copy_(torch.tensor([[40, 90, 17], [33, 64, 9], [39, 41, 10]][i % 3], dtype=torch.int32))
        args[3].fill_([100, 0, 37][i % 3])
        graph, outs = graphs[i % 2]
        state["prefix"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, prefix = [x.clone() for x in outs], state["prefix"].clone()
        state["prefix"].zero_()
        want = serve(own, shared, q, args, kw, to, state, None)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(prefix, state["prefix"])


@pytest.mark.parametrize("q8", [False, True])
def test_graph_large(device, q8):
    """The same of sizes that are cut: pieces of a prefix, rows of the weights over several workgroups, long
    rows of the eviction; replays between eager calls of the same sizes."""
    own = Cache([9000, 700], 2, 64, 64, BF16, q8, news=[600, 300])
    shared = Cache([3001], 2, 64, 64, BF16, q8, seed=1)
    args, kw = on(device, own, shared)
    k, v, ptable, plens, table, lens = args
    ks = {"k_scale": kw["k_scale"]} if q8 else {}
    cu = own.cu.to(device)
    q = torch.randn(900, 8, 64, generator=torch.Generator().manual_seed(5)).bfloat16().to(device)
    to = torch.full((2, 100), -1, dtype=torch.int32, device=device)  # (rows are dropped: weights and lens count)

    def run():
        o, lse = fa.flash_attention_paged_prefix(q, *args, cu_seqlens=cu, return_lse=True, **kw)
        w = fa.paged_attention_weights(q, lse, k, table, lens, cu_seqlens=cu, **ks)
        return (o, lse, w, *fa.paged_cache_evict(k, v, table, lens, w, to, 6000, 500, **kw))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        lens.copy_(torch.tensor([[9000, 700], [8300, 300], [600, 650], [8999, 301]][i], dtype=torch.int32))
        plens.fill_([3001, 17, 0, 2900][i])
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)
        want = run()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)


def test_calls_at_once(device):
    """On several streams at once, each with its own cache, sizes that are cut among them."""
    settings = [Cache([9000 - 700 * i, 300], 2, 64, 64, BF16, i % 2 == 1, seed=i, news=[200 + i, 1]) for i in range(4)]
    shared = [Cache([2000 + i], 2, 64, 64, BF16, i % 2 == 1, seed=9 + i) for i in range(4)]
    on_device = [on(device, o, s) for o, s in zip(settings, shared)]
    qs = [torch.randn(sum(o.news), 4, 64, generator=torch.Generator().manual_seed(i)).bfloat16().to(device)
          for i, o in enumerate(settings)]
    cus, to = [o.cu.to(device) for o in settings], torch.full((2, 60), -1, dtype=torch.int32, device=device)

    def run(i):
        args, kw = on_device[i]
        ks = {"k_scale": kw["k_scale"]} if kw else {}
        o, lse = fa.flash_attention_paged_prefix(qs[i], *args, cu_seqlens=cus[i], return_lse=True, **kw)
        w = fa.paged_attention_weights(qs[i], lse, args[0], *args[4:], cu_seqlens=cus[i], **ks)
        return (o, lse, w, *fa.paged_cache_evict(*args[:2], *args[4:], w, to, 3700, 100, **kw))

    alone = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(4):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        for x, y in zip(alone, got):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_prefix_groups_that_overlap(device):
    """cu_prefix that falls again and again makes more units than there are records: what is written is not
    said, but nothing outside the rows is, and the call ends."""
    own, shared = Cache([20] * 64, 2, 64, 16, FP16, False), Cache([200], 2, 64, 16, FP16, False, seed=3)
    k, v, ptable, plens, table, lens = on(device, own, shared)[0]
    for count in (700, 5000):
        cu = torch.tensor(([0, 64] * count)[:count + 1], dtype=torch.int32, device=device)
        room = torch.full((192, 8, 64), 7.0, dtype=FP16, device=device)
        q = torch.randn(64, 8, 64, dtype=FP16, device=device)
        fa.flash_attention_paged_prefix(q, k, v, ptable.expand(count, -1).contiguous(), plens.expand(count).contiguous(),
                                        table, lens, cu_prefix=cu, out=room[64:128])
        assert (room[:64] == 7).all() and (room[128:] == 7).all()


def test_pools_past_32_bits(device):
    """Pages, codes and scales whose byte offsets pass 2^32."""
    pages, page, hkv, d = 300000, 64, 4, 64
    for dtype in (torch.float8_e4m3fn, FP16):
        q8 = dtype != FP16
        own, shared = Cache([150, 100], hkv, d, page, FP16, q8, news=[90, 1]), Cache([130], hkv, d, page, FP16, q8, seed=2)
        k = torch.empty(pages, hkv, page, d, dtype=dtype, device=device)
        v = torch.empty_like(k)
        kw = {}
        if q8:
            kw = {n: torch.empty(pages, hkv, page, dtype=torch.float8_e8m0fnu, device=device) for n in ("k_scale", "v_scale")}
        assert k.numel() * k.element_size() > 2 ** 32
        where = {}
        for i, c in enumerate((own, shared)):
            for b in range(len(c.lens)):
                for j in range(-(-c.lens[b] // page)):
                    p, to = int(c.table[b, j]), pages - 1 - 1000 * len(where)
                    where[i, p] = to
                    k[to], v[to] = c.k[p].to(device), c.v[p].to(device)
                    if q8:
                        kw["k_scale"].view(torch.uint8)[to] = c.ks.view(torch.uint8)[p].to(device)
                        kw["v_scale"].view(torch.uint8)[to] = c.vs.view(torch.uint8)[p].to(device)
                    c.table[b, j] = to
            c.pages = pages
        table, lens, cu = own.table.to(device), own.seq_lens.to(device), own.cu.to(device)
        q = torch.randn(91, 8, d, generator=torch.Generator().manual_seed(8)).half()
        o, lse = fa.flash_attention_paged_prefix(q.to(device), k, v, shared.table.to(device), shared.seq_lens.to(device),
                                                 table, lens, cu_seqlens=cu, return_lse=True, **kw)
        want, _, tol, _ = ref.attention(con.Joined(own, shared, [0, 0]), q)
        ref.check(o, want, tol * (1 + 2.0 ** -4), "O")
        want, tol = con.weights(own, q, lse.cpu())
        ks = {"k_scale": kw["k_scale"]} if q8 else {}
        for hint in (1, None):
            w = fa.paged_attention_weights(q.to(device), lse, k, table, lens, cu_seqlens=cu, max_query_len=hint, **ks)
            ref.check(w, want, tol, "weights")
        to = torch.tensor([[pages - 2], [pages - 3]], dtype=torch.int32, device=device)
        got, left = fa.paged_cache_evict(k, v, table, lens, w, to, 40, 3, **kw)
        assert got.tolist() == [40, 40]
        for b in range(2):
            for h in range(hkv):
                at = con.stays(w[b, h].tolist(), own.held(b).tolist(), own.lens[b], 40, 3)
                rows = k[int(to[b, 0]), h, :40].double()
                if q8:
                    rows = rows * kw["k_scale"][int(to[b, 0]), h, :40].double()[:, None]
                assert torch.equal(rows.cpu(), own.rows[b][0][h, at]) and torch.equal(left[b, h, :40], w[b, h, at])
        del k, v, kw
        torch.cuda.empty_cache()


def test_workspaces_of_the_c_calls(device):
    """Weights without a workspace (no unit is cut) and prefixes with no more than the states' share of one (own
    keys are not cut) give the same within the same bounds."""
    import ctypes

    from capi_types import LIB
    from test_paged_context_cpu import PagedPrefix, WeighParams
    from test_paged_cpu import PagedCache, PagedParams

    lib = ctypes.CDLL(LIB)
    lib.fa_sm75_last_error.restype = ctypes.c_char_p
    P = ctypes.POINTER
    lib.fa_sm75_paged_weigh.argtypes = [P(WeighParams)]
    lib.fa_sm75_paged_prefix_forward.argtypes = [P(PagedParams), P(PagedPrefix)]
    own, shared = Cache([2500, 33], 2, 64, 64, BF16, False, news=[200, 1]), Cache([700], 2, 64, 64, BF16, False, seed=3)
    k, v, ptable, plens, table, lens = on(device, own, shared)[0]
    q, cu = torch.randn(201, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16(), own.cu.to(device)
    qd = q.to(device)
    c = PagedCache(k=k.data_ptr(), v=v.data_ptr(), block_table=table.data_ptr(), seq_lens=lens.data_ptr(), batch=2, heads_kv=2,
                   head_dim=64, num_pages=k.shape[0], page_size=64, max_pages=table.shape[1], block_table_stride=table.stride(0))
    for t, x in (("k", k), ("v", v)):
        for i, n in enumerate("phn"):
            setattr(c, f"{t}_stride_{n}", x.stride(i))
    x = PagedPrefix(block_table=ptable.data_ptr(), lens=plens.data_ptr(), count=1, max_pages=ptable.shape[1],
                    block_table_stride=ptable.shape[1])
    o, lse = torch.empty_like(qd), torch.empty(8, 201, device=device)
    work = torch.empty(1 << 26, dtype=torch.uint8, device=device)
    p = PagedParams(cache=ctypes.pointer(c), q=qd.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(), tokens=201, heads_q=8,
                    q_stride_t=512, q_stride_h=64, o_stride_t=512, o_stride_h=64, cu_seqlens=cu.data_ptr(), scale=0.125,
                    causal=2, dtype=1, stream=torch.cuda.current_stream().cuda_stream, workspace=work.data_ptr())
    assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(p), ctypes.byref(x)) == 1
    p.workspace_bytes = int(lib.fa_sm75_last_error().split(b"hold ")[1].split(b" ")[0])  # the least
    assert p.workspace_bytes < work.numel()
    work[p.workspace_bytes:] = 77
    assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(p), ctypes.byref(x)) == 0, lib.fa_sm75_last_error()
    assert (work[p.workspace_bytes:] == 77).all()
    want, want_lse, tol, lse_tol = ref.attention(con.Joined(own, shared, [0, 0]), q)
    ref.check(o, want, tol * (1 + 2.0 ** -4), "O")
    ref.check(lse, want_lse, lse_tol + 2.0 ** -15, "LSE")
    # Few rows and short tables: one launch, which needs none.
    p.cu_seqlens, p.tokens, p.workspace, p.workspace_bytes = 0, 2, 0, 0
    assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(p), ctypes.byref(x)) == 0, lib.fa_sm75_last_error()
    ones = Cache([2500, 33], 2, 64, 64, BF16, False, news=[1, 1])
    want, want_lse2, tol, lse_tol = ref.attention(con.Joined(ones, shared, [0, 0]), q[:2])
    ref.check(o[:2], want, tol * (1 + 2.0 ** -4), "O of single tokens")
    ref.check(lse.flatten()[:16].view(8, 2), want_lse2, lse_tol + 2.0 ** -15, "LSE of single tokens")
    lse.copy_(want_lse.float())
    weights = torch.empty(2, 2, 2560, device=device)
    w = WeighParams(cache=ctypes.pointer(c), q=qd.data_ptr(), lse=lse.data_ptr(), weights=weights.data_ptr(),
                    weights_stride_b=5120, weights_stride_h=2560, max_len=2560, tokens=201, heads_q=8, q_stride_t=512,
                    q_stride_h=64, cu_seqlens=cu.data_ptr(), scale=0.125, causal=2, dtype=1, stream=p.stream)
    c.v = 0  # not looked at
    assert lib.fa_sm75_paged_weigh(ctypes.byref(w)) == 0, lib.fa_sm75_last_error()
    want, tol = con.weights(own, q, lse.cpu())
    ref.check(weights, want, tol, "weights")


@pytest.mark.parametrize("seed", range(12))
def test_drawn(device, seed):
    """Drawn sizes, tables, hints and types of all three operators."""
    import random
    rng = random.Random(seed)
    d, page, q8 = rng.choice([64, 128]), rng.choice([16, 32, 128]), rng.random() < 0.5
    hkv = rng.choice([1, 2, 3, 8])
    hq, dtype = hkv * rng.choice([1, 2, 4, 7]), rng.choice([FP16, BF16])
    b = rng.randint(1, 6)
    lens = [rng.choice([0, 1, rng.randint(1, 60), rng.randint(1, 700)]) for _ in range(b)]
    news = [rng.choice([0, 1, min(n, rng.randint(0, 90))]) for n in lens]
    if sum(news) == 0:
        news[0] = 1
    gone = [(i, j) for i, n in enumerate(lens) for j in range(-(-n // page)) if rng.random() < 0.1]
    own = Cache(lens, hkv, d, page, dtype, q8, news=news, seed=seed, gone=gone)
    g = rng.randint(1, 3)
    shared = Cache([rng.randint(0, 900) for _ in range(g)], hkv, d, page, dtype, q8, seed=seed + 100)
    cu = sorted(rng.randint(0, b) for _ in range(g + 1))
    causal = rng.random() < 0.7
    attend(own, shared, cu, device, hq, causal=causal, seed=seed)
    weigh(own, device, hq, causal=causal, seed=seed)
    keep = rng.randint(0, 300)
    evict(own, device, keep, rng.randint(0, keep), seed=seed)
