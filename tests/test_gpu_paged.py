"""The paged cache on the GPU against plain 64-bit references: writing, reading back, and
attention over it, at the sizes, tables and masks where they can go wrong."""
import math

import pytest
import torch

import flash_attention_sm75 as fa
import paged_ref as ref
from paged_ref import Cache

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def attend(c, device, hq, seed=1, causal=True, scale=None, strided=False, one=None, **kw):
    """Runs the call on a cache, as the kernel for few and the one for many new tokens a
    sequence take it, and checks O and LSE; returns the last."""
    g = torch.Generator().manual_seed(seed)
    t = sum(c.news)
    q = torch.randn(t, hq, c.d, generator=g).to(c.dtype)
    args, scales = c.args(device, strided)
    one = all(n == 1 for n in c.news) if one is None else one
    want, want_lse, tol, lse_tol = ref.attention(c, q, causal, scale)
    hints = [kw.pop("max_query_len")] if "max_query_len" in kw else [None] if one else [1, 10 ** 6]
    for hint in hints:
        o, lse = fa.flash_attention_paged(q.to(device), *args, cu_seqlens=None if one else c.cu.to(device),
                                          causal="bottom_right" if causal else False, scale=scale,
                                          return_lse=True, max_query_len=hint, **scales, **kw)
        ref.check(o, want, tol, f"O (max_query_len={hint})")
        ref.check(lse, want_lse, lse_tol, f"LSE (max_query_len={hint})")
    return o, lse


# ---- attention ------------------------------------------------------------------


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens(device, d, dtype, q8, page):
    """One token of each sequence: lengths around tiles and pages, empty ones among them."""
    c = Cache([1, 0, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 300, 1000], 2, d, page, dtype, q8)
    attend(c, device, 8)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (14, 2), (12, 12), (32, 8), (15, 3), (40, 2), (16, 16)])
@pytest.mark.parametrize("q8", [False, True])
def test_heads(device, hq, hkv, q8):
    """Groups of 1 to 20 query heads, KV heads that divide the eight XCDs and do not."""
    attend(Cache([77, 300, 5], hkv, 64, 16, BF16, q8), device, hq)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news", [[4, 4, 4], [1, 9, 2], [0, 3, 0], [70, 5, 33], [130, 1, 257]])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(device, d, q8, news, causal):
    """Several new tokens a sequence, none in some; the chunk can be the whole sequence."""
    lens = [max(n, x) for n, x in zip(news, [130, 200, 257])]
    attend(Cache(lens, 2, d, 16, FP16, q8, news=news), device, 6, causal=causal)


def test_more_new_tokens_than_keys(device):
    """seq_lens below the new tokens' count: the first tokens see no key and get zeros, LSE -inf."""
    c = Cache([3, 0, 40], 2, 64, 16, BF16, False, news=[5, 2, 41])
    o, lse = attend(c, device, 4)
    assert (o[:2] == 0).all() and (lse[:, :2] == -math.inf).all()
    assert (o[5:7] == 0).all() and (o[7] == 0).all()


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("q8", [False, True])
def test_long(device, page, q8):
    """Keys split over many workgroups, one long sequence among short ones."""
    attend(Cache([9000, 3, 2500, 64], 2, 128, page, BF16, q8), device, 8)
    attend(Cache([5000, 3, 1500, 64], 2, 128, page, BF16, q8, news=[40, 2, 1, 64]), device, 8)


def test_one_long_sequence_few_heads(device):
    attend(Cache([20011], 1, 64, 16, FP16, True), device, 7)
    attend(Cache([20011], 1, 64, 16, FP16, True, news=[19]), device, 7)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q8", [False, True])
def test_many_blocks(device, d, q8):
    """More units than the GPU runs at once (none is cut), and one batch of few and of many."""
    attend(Cache([700, 650, 300], 8, d, 64, BF16, q8, news=[700, 1, 300]), device, 32, max_query_len=700)
    attend(Cache([1500, 65], 1, d, 32, FP16, q8, news=[190, 65]), device, 2, max_query_len=190)


@pytest.mark.parametrize("d,q8", [(64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("batch", [1, 2, 5, 33])
def test_equal_lengths(device, d, q8, batch):
    """Sequences of one length: cut into equal pieces each where that suits, whatever the
    number of tiles, and along the line else."""
    for keys in (31, 257, 320, 385, 600, 1025, 2100):
        n = min(keys, max(1, 140 // batch))
        c = Cache([keys] * batch, 2, d, 16, BF16, q8, news=[n] * batch, seed=keys)
        attend(c, device, 6, seed=keys)
        attend(c, device, 6, seed=keys, causal=False)
    c = Cache([4097] * min(batch, 5), 2, d, 16, BF16, q8)
    attend(c, device, 8)


@pytest.mark.parametrize("d", [64, 128])
def test_one_long_unit_among_short_ones(device, d):
    """Units enough that each is merged by its last workgroup, the longest many times the others."""
    c = Cache([9000] + [70] * 40, 1, d, 64, BF16, False, news=[300] + [70] * 40)
    attend(c, device, 8)
    c = Cache([33] * 3 + [6000], 2, d, 16, FP16, True, news=[33] * 3 + [1200])
    attend(c, device, 8)


@pytest.mark.parametrize("d,q8,dtype", [(64, False, FP16), (64, True, BF16), (128, False, BF16), (128, True, FP16)])
def test_wide_tables(device, d, q8, dtype):
    """Tables with room for many more keys than there are: the same kernels, V read past the caches."""
    lens, news = [700, 90, 1, 300, 2000], [20, 9, 1, 0, 32]
    pages = (512 << 20) // (len(lens) * 2 * 2 * d * (1 if q8 else 2)) // 16
    c = Cache(lens, 2, d, 16, dtype, q8, news=news, width=pages)
    attend(c, device, 8, max_query_len=32)


def test_unequal_lengths_of_equal_tiles(device):
    c = Cache([385, 400, 448, 447], 1, 128, 16, FP16, False, news=[40, 1, 448, 3])
    attend(c, device, 4)


@pytest.mark.parametrize("q8", [False, True])
def test_missing_pages(device, q8):
    """Entries that name no page hide their keys: -1, past the pool, the type's limits."""
    c = Cache([500, 100, 40, 33], 2, 64, 16, FP16, q8, news=[3, 1, 2, 1],
              gone=[(0, i) for i in range(9)] + [(1, 6), (2, 0), (2, 1), (2, 2)])
    bad = [c.k.shape[0], 2 ** 31 - 1, -2 ** 31, -7]
    for i, x in zip((3, 4, 5, 6), bad):
        c.table[0, i] = x
    o, lse = attend(c, device, 4)
    assert (o[4:6] == 0).all() and (lse[:, 4:6] == -math.inf).all()  # no page of sequence 2 is left


def test_length_past_the_table(device):
    """seq_lens larger than the table has room for: the keys past it are in no page."""
    c = Cache([100, 90], 2, 64, 16, FP16, False, news=[2, 1], width=3)
    attend(c, device, 4)
    c.seq_lens[1] = 2 ** 31 - 1  # as far as the type goes: every key of the table is seen
    c.lens[1] = 48
    c.rows[1] = [x[:, :48] for x in c.rows[1]]
    (args, kw), q = c.args(device), torch.randn(3, 4, 64).half()
    o = fa.flash_attention_paged(q.to(device), *args, cu_seqlens=c.cu.to(device), **kw)
    want, _, tol, _ = ref.attention(c, q)
    ref.check(o[2:], want[2:], tol[2:], "O")


def test_shared_pages(device):
    """Sequences that share a prefix's pages."""
    c = Cache([96, 96, 50], 2, 64, 16, BF16, True)
    c.table[1, :4] = c.table[0, :4]
    for x in range(2):
        c.rows[1][x][:, :64] = c.rows[0][x][:, :64]
    attend(c, device, 6)


@pytest.mark.parametrize("q8", [False, True])
def test_strided(device, q8):
    """[pages, page, H, D] storage, Q a slice of a wider projection, O written in place."""
    c = Cache([50, 129], 2, 64, 32, FP16, q8, news=[5, 20])
    attend(c, device, 4, strided=True)
    (args, kw), g = c.args(device, True), torch.Generator().manual_seed(3)
    wide = torch.randn(25, 12, 64, generator=g).half().to(device)
    out = torch.full((25, 6, 64), 5.0, dtype=FP16, device=device)
    got = fa.flash_attention_paged(wide[:, 2:6], *args, cu_seqlens=c.cu.to(device), out=out[:, 1:5], **kw)
    assert got.data_ptr() == out[:, 1:5].data_ptr()
    want, _, tol, _ = ref.attention(c, wide[:, 2:6].cpu())
    ref.check(out[:, 1:5], want, tol, "O")
    assert (out[:, 0] == 5).all() and (out[:, 5] == 5).all()


def test_rows_behind_the_last_sequence(device):
    """Rows of Q past cu_seqlens[B] are padding: their O and LSE rows are left as they are."""
    c = Cache([50, 30], 2, 64, 16, FP16, False, news=[3, 1])
    (args, kw), q = c.args(device), torch.randn(9, 4, 64).half()
    q[4:] = math.nan
    out = torch.full((9, 4, 64), 7.0, dtype=FP16, device=device)
    fa.flash_attention_paged(q.to(device), *args, cu_seqlens=c.cu.to(device), out=out, **kw)
    want, _, tol, _ = ref.attention(c, q[:4])
    ref.check(out[:4], want, tol, "O")
    assert (out[4:] == 7).all()


def fused(kind, t, h, d, device):
    """Q and out of one buffer, no element in both."""
    if kind == "halves of every row":
        buf = torch.empty(t, 2 * h, d, dtype=FP16, device=device)
        return buf, buf[:, :h], buf[:, h:]
    if kind == "out first":
        buf = torch.empty(t, 2 * h + 3, d, dtype=FP16, device=device)
        return buf, buf[:, h + 2:2 * h + 2], buf[:, 1:h + 1]
    if kind == "one behind the other":
        buf = torch.empty(2, t, h, d, dtype=FP16, device=device)
        return buf, buf[0], buf[1]
    buf = torch.empty(t, h, 2, d, dtype=FP16, device=device)  # head by head
    return buf, buf[:, :, 1], buf[:, :, 0]


@pytest.mark.parametrize("news", [[5, 20], [1, 0]])
@pytest.mark.parametrize("kind", ["halves of every row", "out first", "one behind the other", "head by head"])
def test_out_beside_q(device, kind, news):
    """out and Q as views of one buffer that share no element of it."""
    c, t = Cache([50, 129], 2, 64, 32, FP16, False, news=news), sum(news)
    (args, kw), g = c.args(device), torch.Generator().manual_seed(3)
    q = torch.randn(t, 4, 64, generator=g).half()
    want, _, tol, _ = ref.attention(c, q)
    buf, at, out = fused(kind, t, 4, 64, device)
    buf.fill_(9.0)
    at.copy_(q)
    got = fa.flash_attention_paged(at, *args, cu_seqlens=c.cu.to(device), out=out, **kw)
    assert got.data_ptr() == out.data_ptr()
    ref.check(out, want, tol, "O")
    assert torch.equal(at.cpu(), q)
    out.fill_(9.0)
    at.fill_(9.0)
    assert (buf == 9).all()


def test_out_beside_the_cache(device):
    """One allocation for the pools and the output."""
    c = Cache([50, 129], 2, 64, 32, FP16, False, news=[5, 20])
    (k, v, table, lens), _ = c.args(device)
    n, q = k.numel(), torch.randn(25, 4, 64).half()
    arena = torch.zeros(2 * n + q.numel(), dtype=FP16, device=device)
    pools = [arena[i * n:(i + 1) * n].view(k.shape) for i in range(2)]
    pools[0].copy_(k)
    pools[1].copy_(v)
    out = arena[2 * n:].view(q.shape)
    fa.flash_attention_paged(q.to(device), *pools, table, lens, cu_seqlens=c.cu.to(device), out=out)
    want, _, tol, _ = ref.attention(c, q)
    ref.check(out, want, tol, "O")


def test_out_that_overlaps_is_refused(device):
    c = Cache([50, 129], 4, 64, 32, FP16, False, news=[5, 20])
    (k, v, table, lens), _ = c.args(device)
    cu = c.cu.to(device)
    buf = torch.zeros(60, 9, 64, dtype=FP16, device=device)
    q = buf[10:35, :4]
    for out in (q, buf[10:35, 1:5], buf[10:35, 3:7], buf[11:36, :4], buf[34:59, 2:6], buf[9:34, 3:7],
                k.view(-1, 4, 64)[:25], v.view(-1, 4, 64)[7:32]):
        with pytest.raises(RuntimeError, match="must not share"):
            fa.flash_attention_paged(q, k, v, table, lens, cu_seqlens=cu, out=out)
    wide = torch.zeros(25, 5, 96, dtype=FP16, device=device)  # rows that overlap in part
    with pytest.raises(RuntimeError, match="must not share"):
        fa.flash_attention_paged(wide[:, :4, :64], k, v, table, lens, cu_seqlens=cu, out=wide[:, :4, 32:])
    flat = torch.zeros(4000 * 64, dtype=FP16, device=device)  # strides of their own
    a = flat.as_strided((25, 4, 64), (512, 64, 1))
    for b in (flat.as_strided((25, 4, 64), (256, 64, 1), 256), flat.as_strided((25, 4, 64), (512, 128, 1), 256)):
        with pytest.raises(RuntimeError, match="must not share"):
            fa.flash_attention_paged(a, k, v, table, lens, cu_seqlens=cu, out=b)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-9, 2.0])
def test_scales(device, scale):
    attend(Cache([200, 10], 2, 64, 16, BF16, False, news=[2, 1]), device, 4, scale=scale)


@pytest.mark.parametrize("news", [[1, 1], [40, 3]])
@pytest.mark.parametrize("q8", [False, True])
def test_nonfinite_rows(device, news, q8):
    """A query's NaN stays in its row (and the pool's unused rows, which hold NaN, reach none)."""
    c = Cache([400, 90], 1, 64, 16, BF16, q8, news=news)
    (args, kw), g = c.args(device), torch.Generator().manual_seed(3)
    t = sum(news)
    q = torch.randn(t, 4, 64, generator=g).bfloat16()
    q[0, 1, 5] = math.nan
    o, lse = fa.flash_attention_paged(q.to(device), *args, cu_seqlens=c.cu.to(device), return_lse=True, **kw)
    want, want_lse, tol, lse_tol = ref.attention(c, q.nan_to_num(0.0))
    assert o[0, 1].isnan().all() and lse[1, 0].isnan()
    keep = torch.ones(t, 4, dtype=torch.bool)
    keep[0, 1] = False
    ref.check(o.cpu()[keep], want[keep], tol[keep], "O")
    ref.check(lse.cpu().T[keep], want_lse.T[keep], lse_tol.T[keep], "LSE")


def test_peaked(device):
    """Scores that keep rising along the keys raise the running maximum again and again."""
    c = Cache([600], 1, 64, 16, FP16, False, news=[3])
    up = torch.linspace(-1, 1, 600)[None, :, None]
    k = (c.rows[0][0] * 0.1 + 12 * up).half()
    for i in range(38):
        p = int(c.table[0, i])
        part = k[:, 16 * i:16 * i + 16]
        c.k[p, :, :part.shape[1]] = part
    c.rows[0][0] = k.double()
    attend(c, device, 4)


def test_max_query_len_is_a_hint(device):
    """Wrong values of it choose another kernel and nothing else."""
    c = Cache([150, 200], 2, 64, 16, BF16, False, news=[60, 1])
    for hint in (1, 5, 60, 61, 10 ** 9, 2 ** 63 - 1):
        attend(c, device, 8, max_query_len=hint)


def test_index_tensors_are_held_to_their_ranges(device):
    """cu_seqlens that falls or passes the rows writes nothing outside them."""
    c = Cache([50, 30], 2, 64, 16, FP16, False, news=[3, 1])
    (args, kw), q = c.args(device), torch.randn(4, 4, 64).half().to(device)
    for cu in ([0, 3, 100], [0, -5, 4], [2 ** 31 - 1, 0, 1], [-2 ** 31, 2, 2 ** 31 - 1], [4, 4, 4]):
        room = torch.full((12, 4, 64), 7.0, dtype=FP16, device=device)
        cu = torch.tensor(cu, dtype=torch.int32, device=device)
        fa.flash_attention_paged(q, *args, cu_seqlens=cu, out=room[4:8], **kw)
        assert (room[:4] == 7).all() and (room[8:] == 7).all()
    lens = torch.tensor([-5, -2 ** 31], dtype=torch.int32, device=device)
    o = fa.flash_attention_paged(q, *args[:3], lens, cu_seqlens=c.cu.to(device), **kw)
    assert (o == 0).all()


@pytest.mark.parametrize("batch,most", [(4096, 1), (9000, 1)])
def test_overlapping_sequences_past_32_bits(device, batch, most):
    """cu_seqlens that falls again and again makes more tiles than 32 bits count: what is
    written is not said, but nothing outside the rows is, and the call ends."""
    page, keys = 1 << 15, 1 << 23
    k = torch.zeros(1, 1, page, 64, dtype=torch.float8_e4m3fn, device=device)
    s = torch.full((1, 1, page), 127, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    table = torch.zeros(1, keys // page, dtype=torch.int32, device=device).expand(batch, -1).contiguous()
    lens = torch.full((batch,), keys, dtype=torch.int32, device=device)
    cu = torch.tensor(([0, 64] * batch)[:batch + 1], dtype=torch.int32, device=device)
    room = torch.full((192, 1, 64), 7.0, dtype=FP16, device=device)
    q = torch.randn(64, 1, 64, dtype=FP16, device=device)
    fa.flash_attention_paged(q, k, k.clone(), table, lens, cu_seqlens=cu, k_scale=s, v_scale=s,
                             out=room[64:128], max_query_len=most)
    assert (room[:64] == 7).all() and (room[128:] == 7).all()


def test_nothing_to_do(device):
    c = Cache([5], 2, 64, 16, FP16, False)
    args, _ = c.args(device)
    empty = torch.empty(0, 4, 64, dtype=FP16, device=device)
    cu = torch.zeros(2, dtype=torch.int32, device=device)
    assert fa.flash_attention_paged(empty, *args, cu_seqlens=cu).shape == (0, 4, 64)
    none = (args[0], args[1], args[2][:0], args[3][:0])
    assert fa.flash_attention_paged(empty, *none).shape == (0, 4, 64)
    out = torch.full((2, 4, 64), 3.0, dtype=FP16, device=device)
    fa.flash_attention_paged(torch.zeros_like(out), *none, cu_seqlens=cu[:1], out=out)
    assert (out == 3).all()
    pool = (args[0][:0], args[1][:0], args[2], args[3])  # a pool without pages
    o, lse = fa.flash_attention_paged(torch.ones(1, 4, 64, dtype=FP16, device=device), *pool, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()


def test_same_bits_every_time(device):
    c = Cache([3000, 17, 900], 2, 128, 16, BF16, True, news=[2, 1, 3])
    first = attend(c, device, 8)
    for _ in range(3):
        again = attend(c, device, 8)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---- writing and reading ---------------------------------------------------------


def written(c, device, k, v, cu, strided=False):
    """The pools after a write over a NaN pool, as CPU tensors."""
    (kc, vc, table, lens), kw = c.args(device, strided)
    fa.paged_cache_write(k.to(device), v.to(device), kc, vc, table, lens, cu_seqlens=cu, **kw)
    return [x.cpu() for x in (kc, vc, *kw.values())]


def same(a, b):
    a, b = (x.view(torch.uint8) if x.dtype == torch.float8_e8m0fnu else x.float() for x in (a, b))
    return torch.equal(a.nan_to_num(123.0), b.nan_to_num(123.0)) if a.is_floating_point() else torch.equal(a, b)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_write(device, d, q8, dtype, strided):
    """New rows arrive where the table says, everything else stays."""
    news = [3, 0, 40, 1, 5]
    c = Cache([20, 9, 77, 1, 3], 3, d, 16, dtype, q8, news=news, gone=[(2, 3)])
    g = torch.Generator().manual_seed(9)
    k, v = ((torch.randn(sum(news) + 2, 3, d, generator=g) * 3).to(dtype) for _ in "kv")
    want = [x.clone() for x in (c.k, c.v, *((c.ks, c.vs) if q8 else ()))]
    for b, n in enumerate(news):
        for i in range(n):
            pos, row = c.lens[b] - n + i, int(c.cu[b]) + i
            if pos < 0 or c.table[b, pos // 16] < 0:
                continue
            p, r = int(c.table[b, pos // 16]), pos % 16
            for x, new in enumerate((k, v)):
                if q8:
                    codes, scale = ref.quantise(new[row])
                    want[x][p, :, r] = codes
                    want[2 + x].view(torch.uint8)[p, :, r] = scale.view(torch.uint8)
                else:
                    want[x][p, :, r] = new[row]
    for got, w in zip(written(c, device, k, v, c.cu.to(device), strided), want):
        assert same(got, w)


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_write_extremes(device, dtype):
    """Rows of zeros, infinities, NaN, the type's limits, and every border of the scale."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    rows = [[0.0], [math.inf, 1.0], [math.nan, 3.0], [math.inf], [-math.inf, math.nan, top], [top], [-top],
            [tiny], [tiny, -3 * tiny], [448.0], [449.0], [448.0 * 2, 1], [450.0 * 2], [0.4375], [0.438],
            [57344.0, 65280.0 if dtype == FP16 else 3e38], [1.0, 2.0 ** -9, 2.0 ** -10, 2.0 ** -11, 3 * 2.0 ** -11],
            [17.0, 18.0, 19.0, 21.0, 27.0, 29.0, 256.0]]
    x = torch.zeros(len(rows), 1, 64)
    for i, r in enumerate(rows):
        x[i, 0, :len(r)] = torch.tensor(r, dtype=torch.float64).float()
    x = x.to(dtype)
    c = Cache([len(rows)], 1, 64, 32, dtype, True, news=[len(rows)])
    k, v, ks, vs = written(c, device, x, -x, c.cu.to(device))
    codes, scale = ref.quantise(x[:, 0])
    p = int(c.table[0, 0])
    assert same(k[p, 0, :len(rows)], codes) and same(ks[p, 0, :len(rows)], scale)
    assert same(vs[p, 0, :len(rows)], scale)
    # and back: exact 16-bit numbers
    dev = [t.to(device) for t in (k, v, c.table, c.seq_lens)]
    kr, _ = fa.paged_cache_read(*dev, max_len=len(rows), k_scale=ks.to(device), v_scale=vs.to(device), dtype=dtype)
    want = codes.double() * scale.double()[:, None]
    assert torch.equal(kr[0, 0].double().cpu().nan_to_num(9.9), want.nan_to_num(9.9))


def test_write_single_tokens(device):
    """Without cu_seqlens row b is sequence b's token; K and V as views of one projection."""
    c = Cache([1, 16, 17, 0, 33], 2, 64, 16, BF16, False)
    qkv = torch.randn(5, 3, 2, 64).bfloat16()
    before = c.k.clone()
    k, v = written(c, device, qkv[:, 1], qkv[:, 2], None)
    for b, n in enumerate(c.lens):
        if n:
            p, r = int(c.table[b, (n - 1) // 16]), (n - 1) % 16
            before[p, :, r] = qkv[b, 1]
            assert torch.equal(v[p, :, r], qkv[b, 2])
    assert same(k, before)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("q8,dtype", [(False, FP16), (False, BF16), (True, FP16), (True, BF16)])
@pytest.mark.parametrize("d", [64, 128])
def test_read(device, d, q8, dtype, strided):
    c = Cache([20, 0, 77, 1, 129], 3, d, 32, dtype, q8, gone=[(2, 0), (4, 2)])
    args, kw = c.args(device, strided)
    for max_len in (None, 1, 80, 200):
        k, v = fa.paged_cache_read(*args, max_len=max_len, dtype=dtype if q8 else None, **kw)
        longest = c.width * 32 if max_len is None else max_len
        assert k.shape == (5, 3, longest, d) and k.dtype == dtype
        for b, n in enumerate(c.lens):
            held = c.held(b)
            for got, rows in ((k, c.rows[b][0]), (v, c.rows[b][1])):
                want = torch.zeros(3, longest, d, dtype=torch.float64)
                m = min(n, longest)
                want[:, :m] = torch.where(held[:m, None], rows[:, :m], 0.0)
                assert torch.equal(got[b].double().cpu(), want)


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_read_every_code_and_scale(device, dtype):
    """Any code times any scale, also ones that no write leaves: rounded to the type, NaN for byte 255."""
    code = torch.arange(1024) % 4 * 64 + torch.arange(64)[:, None]
    codes = code.T.to(torch.uint8).reshape(1, 1, 1024, 64).contiguous().view(torch.float8_e4m3fn)
    byte = (torch.arange(1024) // 4).to(torch.uint8)
    scale = byte.reshape(1, 1, 1024).view(torch.float8_e8m0fnu)
    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    lens = torch.tensor([1024], dtype=torch.int32, device=device)
    k, v = fa.paged_cache_read(codes.to(device), codes.to(device), table, lens, k_scale=scale.to(device),
                               v_scale=scale.to(device), dtype=dtype)
    factor = torch.exp2(byte.double() - 127).masked_fill(byte == 255, math.nan)
    want = (codes[0, 0].float().double() * factor[:, None]).to(dtype)
    for got in (k, v):
        assert torch.equal(got[0, 0].cpu().nan_to_num(nan=-1.5), want.nan_to_num(nan=-1.5))


def test_read_nothing(device):
    c = Cache([5, 3], 2, 64, 16, FP16, False)
    args, _ = c.args(device)
    assert fa.paged_cache_read(*args, max_len=0)[0].shape == (2, 2, 0, 64)
    k, v = fa.paged_cache_read(args[0][:0], args[1][:0], *args[2:], max_len=20)
    assert k.shape == (2, 2, 20, 64) and (k == 0).all() and (v == 0).all()


@pytest.mark.parametrize("batch,hkv", [(2100, 64), (2, 1 << 16)])
@pytest.mark.parametrize("q8", [False, True])
def test_read_many_sequences_and_heads(device, q8, batch, hkv):
    """More heads of sequences than a dimension of the grid holds (65535)."""
    d, page, max_len = 64, 16, 5
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(2, hkv, page, d, generator=g).half() for _ in "kv")
    kw = {}
    if q8:
        k, v = (x.float().to(torch.float8_e4m3fn) for x in (k, v))
        kw = {n: torch.randint(120, 130, (2, hkv, page), generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)
              for n in ("k_scale", "v_scale")}
    table = torch.randint(-1, 2, (batch, 1), generator=g, dtype=torch.int32)
    lens = torch.randint(0, 8, (batch,), generator=g, dtype=torch.int32)
    got = fa.paged_cache_read(k.to(device), v.to(device), table.to(device), lens.to(device), max_len=max_len,
                              dtype=FP16, **{n: x.to(device) for n, x in kw.items()})
    pos = torch.arange(max_len)
    held = (pos < lens[:, None]) & (table >= 0)
    for out, pool, scale in zip(got, (k, v), ("k_scale", "v_scale")):
        want = pool[:, :, :max_len].float()
        if q8:  # (exact in binary16)
            want = want * kw[scale][:, :, :max_len].float()[..., None]
        want = want.half()[table[:, 0].clamp(min=0).long()]
        want.masked_fill_(~held[:, None, :, None], 0.0)
        assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("q8", [False, True])
def test_what_is_written_counts_as_changed(device, q8):
    """Autograd sees the writes: versions rise, also a view's base's, and a backward that kept the
    old values raises, as after torch's own in-place operations."""
    c = Cache([20, 9], 2, 64, 16, FP16, q8, news=[3, 1])
    (k, v, table, lens), kw = c.args(device)
    new = torch.randn(4, 2, 64, device=device).half()
    changed = [k, v, *kw.values()]
    before = [x._version for x in changed]
    w = torch.ones((), device=device, requires_grad=True)
    loss = (w * k.float().nan_to_num(0.0)).sum() if q8 else (w.half() * k).sum()  # the 16-bit pool is kept
    fa.paged_cache_write(new, new, k, v, table, lens, cu_seqlens=c.cu.to(device), **kw)
    assert all(x._version > n for x, n in zip(changed, before))
    if q8:
        loss.backward()  # (a copy was kept)
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = [x._version for x in changed]
    q = torch.randn(4, 6, 64, device=device).half()
    wide = torch.zeros(4, 8, 64, dtype=FP16, device=device)
    version = wide._version
    fa.flash_attention_paged(q, k, v, table, lens, cu_seqlens=c.cu.to(device), out=wide[:, 1:7], **kw)
    assert wide._version > version and q._version == 0
    fa.paged_cache_read(k, v, table, lens, dtype=FP16, **kw)
    assert [x._version for x in changed] == before


def test_inference_tensors(device):
    """A cache and an output made in inference mode, used in it and outside of it."""
    c = Cache([20, 9], 2, 64, 16, FP16, False, news=[3, 1])
    with torch.inference_mode():
        (k, v, table, lens), _ = c.args(device)
        out = torch.zeros(4, 4, 64, dtype=FP16, device=device)
    cu, new = c.cu.to(device), torch.randn(4, 2, 64, device=device).half()
    got = []
    for mode in (torch.inference_mode, torch.no_grad, torch.enable_grad):
        with mode():
            fa.paged_cache_write(new, new, k, v, table, lens, cu_seqlens=cu)
            fa.flash_attention_paged(new.repeat(1, 2, 1), k, v, table, lens, cu_seqlens=cu, out=out)
        got.append((k.cpu(), out.cpu()))
    for pool, o in got[1:]:
        assert same(pool, got[0][0]) and torch.equal(o, got[0][1])


# ---- together ----------------------------------------------------------------------


@pytest.mark.parametrize("q8", [False, True])
def test_a_batch_grows(device, q8):
    """A serving loop: prompts in chunks, then single tokens; what is read back gives the other
    kernels the same attention."""
    d, hq, hkv, page, dtype = 64, 6, 2, 16, BF16
    g = torch.Generator().manual_seed(5)
    total = [75, 40]
    c = Cache(total, hkv, d, page, dtype, q8, seed=11)  # its tables; the rows come from the writes
    (kc, vc, table, _), kw = c.args(device)
    new = [torch.randn(2, n, hkv, d, generator=g).to(dtype) for n in total]
    done = [0, 0]
    for step in ([30, 17], [33, 20], [1, 1], [1, 1], [10, 0], [0, 1]):
        k, v = (torch.cat([new[b][x, done[b]:done[b] + n] for b, n in enumerate(step)]) for x in range(2))
        done = [a + n for a, n in zip(done, step)]
        lens = torch.tensor(done, dtype=torch.int32, device=device)
        cu = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device=device)
        fa.paged_cache_write(k.to(device), v.to(device), kc, vc, table, lens, cu_seqlens=cu, **kw)
        q = torch.randn(sum(step), hq, d, generator=g).to(dtype)
        o = fa.flash_attention_paged(q.to(device), kc, vc, table, lens, cu_seqlens=cu, **kw)
        kr, vr = fa.paged_cache_read(kc, vc, table, lens, dtype=dtype, **kw)
        for b, n in enumerate(step):
            if n == 0:
                continue
            rows = [ref._through8(x[:done[b]]) if q8 else x[:done[b]].double() for x in new[b]]
            c.rows[b] = [x.transpose(0, 1) for x in rows]
            for got, want in ((kr, rows[0]), (vr, rows[1])):
                assert torch.equal(got[b, :, :done[b]].double().cpu(), want.transpose(0, 1))
                assert (got[b, :, done[b]:] == 0).all()
            part = slice(int(cu[b]), int(cu[b]) + n)
            dense = fa.flash_attention_forward_ex(q[part].to(device).transpose(0, 1)[None],
                                                  kr[b:b + 1, :, :done[b]], vr[b:b + 1, :, :done[b]],
                                                  causal="bottom_right")
            one = Cache([done[b]], hkv, d, page, dtype, False, news=[n])
            one.rows = [c.rows[b]]
            want, _, tol, _ = ref.attention(one, q[part])
            ref.check(o[part], want, tol, f"O of sequence {b}")
            ref.check(dense[0].transpose(0, 1), want, 2 * tol, f"dense O of sequence {b}")


# ---- batches, shapes and tables at large ----------------------------------------------


@pytest.mark.parametrize("hint", [1, 10 ** 6])
@pytest.mark.parametrize("q8", [False, True])
def test_many_sequences(device, q8, hint):
    """More sequences than lanes, empty ones and ones without new tokens among them."""
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 90, (150,), generator=g).tolist()
    news = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 4, (150,), generator=g))]
    lens[140], news[140] = 900, 60
    c = Cache(lens, 2, 64, 16, BF16, q8, news=news)
    attend(c, device, 6, max_query_len=hint)


def test_write_many_sequences(device):
    """The sequence of a row is found among more than 64 of them, many without new rows."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(1, 40, (200,), generator=g).tolist()
    news = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 3, (200,), generator=g))]
    c = Cache(lens, 1, 64, 16, FP16, False, news=news)
    k = torch.randn(sum(news), 1, 64, generator=g).half()
    want = c.k.clone()
    for b, n in enumerate(news):
        for i in range(n):
            pos = lens[b] - n + i
            want[int(c.table[b, pos // 16]), :, pos % 16] = k[int(c.cu[b]) + i]
    got, _ = written(c, device, k, -k, c.cu.to(device))
    assert same(got, want)


@pytest.mark.parametrize("hq,hkv", [(160, 1), (33, 1), (48, 16), (24, 24)])
def test_wide_groups(device, hq, hkv):
    """More query heads to a KV head than a block of either kernel has rows."""
    c = Cache([50, 7], hkv, 64, 16, FP16, True, news=[2, 1])
    attend(c, device, hq)
    attend(Cache([50, 7], hkv, 64, 16, FP16, False), device, hq, max_query_len=1)


@pytest.mark.parametrize("page", [16, 4096])
def test_table_wider_than_needed(device, page):
    """A table with room for far longer sequences, its rows a slice of a wider one."""
    c = Cache([130, 700], 2, 64, page, BF16, False, news=[3, 40])
    (k, v, table, lens), kw = c.args(device)
    wide = torch.full((2, 3000), 2 ** 30, dtype=torch.int32, device=device)
    wide[:, 5:5 + table.shape[1]] = table
    q = torch.randn(43, 4, 64).bfloat16()
    want, _, tol, _ = ref.attention(c, q)
    for hint in (1, 40):
        o = fa.flash_attention_paged(q.to(device), k, v, wide[:, 5:2900], lens, cu_seqlens=c.cu.to(device),
                                     max_query_len=hint, **kw)
        ref.check(o, want, tol, "O")
    kr, _ = fa.paged_cache_read(k, v, wide[:, 5:2900], lens, max_len=710, **kw)
    assert torch.equal(kr[1, :, :700].double().cpu(), c.rows[1][0])


def test_pool_past_32_bits(device):
    """Pages, codes and scales whose byte offsets pass 2^32."""
    pages, page, hkv, d = 300000, 64, 4, 64
    for dtype in (torch.float8_e4m3fn, FP16):
        k = torch.empty(pages, hkv, page, d, dtype=dtype, device=device)
        v = torch.empty_like(k)
        assert k.numel() * k.element_size() > 2 ** 32
        kw = {}
        if dtype == torch.float8_e4m3fn:
            kw = {n: torch.empty(pages, hkv, page, dtype=torch.float8_e8m0fnu, device=device)
                  for n in ("k_scale", "v_scale")}
        table = torch.tensor([[pages - 1, 0, pages - 7], [5, pages // 2, -1]], dtype=torch.int32, device=device)
        c = Cache([150, 100], hkv, d, page, FP16, bool(kw), news=[150, 100])
        c.table, c.pages = table.cpu(), pages
        g = torch.Generator().manual_seed(8)
        new = [torch.randn(250, hkv, d, generator=g).half() for _ in "kv"]
        c.rows = [[(ref._through8(x[p]) if kw else x[p].double()).transpose(0, 1) for x in new]
                  for p in (slice(0, 150), slice(150, 250))]
        lens, cu = c.seq_lens.to(device), c.cu.to(device)
        fa.paged_cache_write(*(x.to(device) for x in new), k, v, table, lens, cu_seqlens=cu, **kw)
        kr, vr = fa.paged_cache_read(k, v, table, lens, dtype=FP16, **kw)
        for b, n in enumerate(c.lens):
            assert torch.equal(kr[b, :, :n].double().cpu(), c.rows[b][0])
            assert torch.equal(vr[b, :, :n].double().cpu(), c.rows[b][1])
        q = torch.randn(250, 8, d, generator=g).half()
        want, _, tol, _ = ref.attention(c, q)
        for hint in (1, 150):
            o = fa.flash_attention_paged(q.to(device), k, v, table, lens, cu_seqlens=cu, max_query_len=hint, **kw)
            ref.check(o, want, tol, "O")
        del k, v, kw, kr, vr
        torch.cuda.empty_cache()


def test_sweep(device):
    """Seeded cases over the sizes, types, layouts and tables that the calls take."""
    import os
    import random

    for seed in range(int(os.environ.get("FA_PAGED_SWEEP_CASES", "60"))):
        r = random.Random(1000 + seed)
        b = r.choice([1, 1, 2, 3, 7, 20])
        lens = [r.choice([0, 1, r.randint(1, 64), r.randint(1, 400), r.randint(1, 1500 if b < 4 else 300)])
                for _ in range(b)]
        kind = r.choice(["one", "few", "chunk", "mixed"])
        most = {"one": 1, "few": 5, "chunk": 300, "mixed": 90}[kind]
        news = [1 if kind == "one" or (kind == "mixed" and r.random() < 0.7) else r.randint(0, most) for _ in lens]
        if kind != "one" and r.random() < 0.7:
            news = [min(n, x) for n, x in zip(news, lens)]
        hkv, group = r.choice([(1, 1), (1, 7), (2, 4), (3, 2), (8, 4), (2, 1), (4, 9)])
        d, dtype, q8, page = r.choice([64, 128]), r.choice([FP16, BF16]), r.random() < 0.5, r.choice([16, 32, 64, 256])
        gone = [(i, r.randrange(-(-n // page))) for i, n in enumerate(lens) if n and r.random() < 0.2]
        if sum(news) == 0:
            continue
        print(f"case {seed}: lens {lens} news {news} hkv {hkv} group {group} d {d} {dtype} q8 {q8} page {page}", flush=True)
        c = Cache(lens, hkv, d, page, dtype, q8, seed=seed, news=news, gone=gone)
        attend(c, device, hkv * group, seed=seed, causal=r.random() < 0.8, strided=r.random() < 0.3)


# ---- streams and graphs ---------------------------------------------------------------


def test_other_streams(device):
    """Calls on streams of their own, at once, each with its own cache; and a cache whose calls
    follow each other on one stream that is not the current one when it is read."""
    caches = [Cache([400 + 50 * i, 33], 2, 64, 16, BF16, i % 2 == 1, seed=i, news=[1 + 20 * (i % 3), 1]) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in caches]
    g = torch.Generator().manual_seed(1)
    qs = [torch.randn(sum(c.news), 6, 64, generator=g).bfloat16() for c in caches]
    on = [(c.args(device), q.to(device), c.cu.to(device)) for c, q in zip(caches, qs)]
    torch.cuda.synchronize()
    outs = [[] for _ in caches]
    for _ in range(5):
        for i, (s, ((args, kw), q, cu)) in enumerate(zip(streams, on)):
            with torch.cuda.stream(s):
                outs[i].append(fa.flash_attention_paged(q, *args, cu_seqlens=cu, max_query_len=21, **kw))
    torch.cuda.synchronize()
    for c, q, o in zip(caches, qs, outs):
        want, _, tol, _ = ref.attention(c, q)
        for x in o:
            ref.check(x, want, tol, "O")
            assert torch.equal(x, o[0])


@pytest.mark.parametrize("most", [1, 70])
@pytest.mark.parametrize("q8", [False, True])
def test_captured(device, q8, most):
    """A captured write, attention and read-back, replayed over tables, lengths and rows that
    change in between, against eager calls, which run between the replays too."""
    hkv, hq, d, page, dtype = 2, 8, 64, 16, FP16
    c = Cache([900, 300, 64], hkv, d, page, dtype, q8, news=[most, 1, 1])
    (k, v, table, lens), kw = c.args(device)
    t = most + 2
    cu = c.cu.to(device)
    new = [torch.randn(t, hkv, d, device=device).to(dtype) for _ in "kv"]
    q = torch.randn(t, hq, d, device=device).to(dtype)
    out = torch.zeros_like(q)

    def calls():
        fa.paged_cache_write(*new, k, v, table, lens, cu_seqlens=cu, **kw)
        fa.flash_attention_paged(q, k, v, table, lens, cu_seqlens=cu, max_query_len=most, out=out, **kw)
        return fa.paged_cache_read(k, v, table, lens, max_len=901, dtype=dtype, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kr, vr = calls()
    g = torch.Generator().manual_seed(6)
    for step in range(4):
        for x in new + [q]:
            x.copy_(torch.randn(x.shape, generator=g))
        lens.copy_(torch.tensor([900 - 37 * step, 300 - 100 * step, 64 - step], dtype=torch.int32))
        rows = torch.randperm(3, generator=g).tolist()
        table.copy_(c.table[rows][:, :])  # whose pages belong to whom
        lens.copy_(torch.minimum(lens.cpu(), torch.tensor([c.lens[i] for i in rows], dtype=torch.int32)))
        state = [x.clone() for x in (k, v, *kw.values())]
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, kr, vr, k, v, *kw.values())]
        for x, y in zip((k, v, *kw.values()), state):
            x.copy_(y)
        out.zero_()
        eager = calls()
        torch.cuda.synchronize()
        for a, b in zip(got, (out, *eager, k, v, *kw.values())):
            assert same(a.cpu(), b.cpu()), step
