"""Shared prefixes, attention weights and eviction without a GPU: refusals of the C ABI and of the Python
calls, sizes, and the references themselves."""
import ctypes
import math

import pytest
import torch

import paged_context_ref as con
import paged_ref as ref
from capi_types import LIB
from paged_ref import Cache
from test_paged_cpu import BAD_CACHES, I64, INT, PTR, PagedCache, PagedParams, cache, params


class PagedPrefix(ctypes.Structure):
    """fa_paged_prefix."""
    _fields_ = [("block_table", PTR), ("lens", PTR), ("count", I64), ("max_pages", I64), ("block_table_stride", I64),
                ("cu_prefix", PTR), ("max_queries", I64)]


class WeighParams(ctypes.Structure):
    """fa_paged_weigh_params."""
    _fields_ = [("cache", ctypes.POINTER(PagedCache)), ("q", PTR), ("lse", PTR), ("weights", PTR),
                ("weights_stride_b", I64), ("weights_stride_h", I64), ("max_len", I64), ("add", INT),
                ("tokens", I64), ("heads_q", I64), ("q_stride_t", I64), ("q_stride_h", I64), ("cu_seqlens", PTR),
                ("max_query_len", I64), ("scale", ctypes.c_float), ("causal", INT), ("dtype", INT), ("stream", PTR),
                ("workspace", PTR), ("workspace_bytes", I64)]


class EvictParams(ctypes.Structure):
    """fa_paged_evict_params."""
    _fields_ = [("cache", ctypes.POINTER(PagedCache)), ("weights", PTR), ("weights_stride_b", I64),
                ("weights_stride_h", I64), ("weights_len", I64), ("to_table", PTR), ("to_pages", I64),
                ("to_table_stride", I64), ("keep", I64), ("recent", I64), ("new_lens", PTR), ("new_weights", PTR),
                ("stream", PTR), ("workspace", PTR), ("workspace_bytes", I64)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.fa_sm75_last_error.restype = ctypes.c_char_p
    P = ctypes.POINTER
    lib.fa_sm75_paged_prefix_forward.argtypes = [P(PagedParams), P(PagedPrefix)]
    lib.fa_sm75_paged_prefix_workspace_size.argtypes = [P(PagedParams), P(PagedPrefix)]
    lib.fa_sm75_paged_workspace_size.argtypes = [P(PagedParams)]
    lib.fa_sm75_paged_weigh.argtypes = lib.fa_sm75_paged_weigh_workspace_size.argtypes = [P(WeighParams)]
    lib.fa_sm75_paged_evict.argtypes = lib.fa_sm75_paged_evict_workspace_size.argtypes = [P(EvictParams)]
    for f in ("prefix", "weigh", "evict"):
        getattr(lib, f"fa_sm75_paged_{f}_workspace_size").restype = I64
    lib.fa_sm75_paged_workspace_size.restype = I64
    return lib


def prefix(**kw):
    x = PagedPrefix(block_table=0x1000, lens=0x1000, count=1, max_pages=4, block_table_stride=4)
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def weigh(c, **kw):
    p = WeighParams(cache=ctypes.pointer(c), q=0x10000, lse=0x1000, weights=0x1000, weights_stride_b=128,
                    weights_stride_h=64, max_len=64, tokens=2, heads_q=4, q_stride_t=256, q_stride_h=64, scale=0.125,
                    causal=2)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def evict(c, **kw):
    p = EvictParams(cache=ctypes.pointer(c), weights=0x1000, weights_stride_b=128, weights_stride_h=64,
                    weights_len=64, to_table=0x1000, to_pages=2, to_table_stride=2, keep=20, recent=3, new_lens=0x1000,
                    new_weights=0x1000, workspace=0x1000, workspace_bytes=1 << 20)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,status,msg", BAD_CACHES)
def test_cache_refusals(lib, kw, status, msg):
    c = cache(**kw)
    if "v" not in kw and not any(k.startswith("v") for k in kw):  # (V is not looked at by weigh)
        assert lib.fa_sm75_paged_weigh(ctypes.byref(weigh(c))) == status or b"go together" in msg
    for call in (lambda: lib.fa_sm75_paged_prefix_forward(ctypes.byref(params(c)), ctypes.byref(prefix())),
                 lambda: lib.fa_sm75_paged_evict(ctypes.byref(evict(c)))):
        assert call() == status
        assert msg in lib.fa_sm75_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(count=-1), 1, b"non-negative"),
    (dict(max_pages=-1), 1, b"non-negative"),
    (dict(block_table_stride=-4), 1, b"non-negative"),
    (dict(max_queries=-1), 1, b"non-negative"),
    (dict(count=(1 << 20) + 1, cu_prefix=0x1000), 5, b"2^20"),
    (dict(max_pages=(1 << 26) + 1), 5, b"2^30 tokens"),
    (dict(lens=0), 1, b"must not be NULL"),
    (dict(block_table=0), 1, b"must not be NULL"),
    (dict(count=2), 1, b"there is one prefix, got 2"),
    (dict(count=0), 1, b"there is one prefix, got 0"),
    (dict(cu_prefix=0x1002), 4, b"4-byte aligned"),
    (dict(lens=0x1001), 4, b"4-byte aligned"),
])
def test_prefix_refusals(lib, kw, status, msg):
    p, x = params(cache()), prefix(**kw)
    assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(p), ctypes.byref(x)) == status
    assert msg in lib.fa_sm75_last_error()
    before = lib.fa_sm75_last_error()
    assert lib.fa_sm75_paged_prefix_workspace_size(ctypes.byref(p), ctypes.byref(x)) == 0
    assert lib.fa_sm75_last_error() == before


def test_prefix_too_many_units(lib):
    x = prefix(count=1 << 20, cu_prefix=0x1000)
    assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(params(cache(heads_kv=8), heads_q=8)), ctypes.byref(x)) == 5
    assert b"prefixes * heads_kv exceeds 2^27" in lib.fa_sm75_last_error()


def test_prefix_workspace(lib):
    """The rows' states at least (a record of 128 rows for each workgroup: of one block of rows of two heads), where
    the prefixes' tables have more room than each sequence would read for itself; without them the call is refused,
    before it asks the device anything."""
    p, x = params(cache()), prefix(max_pages=1 << 20, block_table_stride=1 << 20)
    states = 2 * 128 * (64 + 2) * 4 + 16
    size = lib.fa_sm75_paged_prefix_workspace_size(ctypes.byref(p), ctypes.byref(x))
    assert size >= states and size % 16 == 0
    for kw in (dict(), dict(workspace=0x1000, workspace_bytes=states - 1)):
        assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(params(cache(), **kw)), ctypes.byref(x)) == 1
        assert b"bytes at least, got" in lib.fa_sm75_last_error()
    assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(p), None) == 1
    assert lib.fa_sm75_paged_prefix_forward(None, ctypes.byref(x)) == 1
    none = prefix(count=0, cu_prefix=0x1000)  # no prefix: what the plain call uses
    assert lib.fa_sm75_paged_prefix_workspace_size(ctypes.byref(p), ctypes.byref(none)) == \
        lib.fa_sm75_paged_workspace_size(ctypes.byref(p))
    for kw, pk in ((dict(batch=0), dict(tokens=0)), ({}, dict(tokens=0, cu_seqlens=0x1000)), ({}, dict(heads_q=0))):
        p = params(cache(**kw), q=0, o=0, **pk)
        assert lib.fa_sm75_paged_prefix_forward(ctypes.byref(p), ctypes.byref(x)) == 0
        assert lib.fa_sm75_paged_prefix_workspace_size(ctypes.byref(p), ctypes.byref(x)) == 0


def prefix_call(hq, hkv, d, q8, b, keys, prefix_keys, prefixes=1, page=16):
    """One token of each of b sequences with room for `keys` own ones behind prefixes with room for prefix_keys."""
    c = cache(batch=b, heads_kv=hkv, head_dim=d, page_size=page, max_pages=-(-keys // page), k_stride_n=d, v_stride_n=d,
              block_table_stride=-(-keys // page), **(dict(k_scale=0x1000, v_scale=0x1000) if q8 else {}))
    p = params(c, heads_q=hq, tokens=b)
    x = prefix(count=prefixes, max_pages=-(-prefix_keys // page), cu_prefix=0x1000)
    return p, x


def cut_bytes(rows, d):
    """A plan's records where 512 workgroups run at once."""
    return 512 * 2 * (rows * (d + 2) * 4 + 8) + 16


# Sequences, keys and whether units are left whole: sizes of which both were measured, those apart by 3% or less left out.
OWN_KEYS = [
    (32, 8, 128, False, [(1, 512, True), (2, 1024, False), (8, 512, True), (16, 768, True), (32, 1024, True), (48, 1024, True),
                         (64, 1536, True), (48, 2048, False), (64, 2048, False), (96, 2048, False), (128, 4096, False)]),
    (32, 8, 128, True, [(4, 1536, False), (16, 1024, True), (47, 1504, True), (48, 1504, True), (49, 1504, True),
                        (48, 2048, True), (64, 2048, True), (32, 2048, False), (48, 4096, False), (64, 4096, False)]),
    (14, 2, 64, False, [(4, 512, True), (4, 2048, False), (96, 768, True), (128, 1536, True), (256, 1536, True), (256, 2048, True),
                        (64, 4096, False), (256, 4096, False)]),
]


@pytest.mark.parametrize("hq,hkv,d,q8,sizes", OWN_KEYS)
def test_prefix_own_keys_cut_or_whole(lib, hq, hkv, d, q8, sizes):
    """Behind a prefix, units of the own keys are cut where that was measured to be faster, and no workspace is asked
    for where they are not: the border rises with the share of the GPU that the units fill."""
    for b, keys, whole in sizes:
        p, x = prefix_call(hq, hkv, d, q8, b, keys, 1 << 20)
        size = lib.fa_sm75_paged_prefix_workspace_size(ctypes.byref(p), ctypes.byref(x))
        states = (size - cut_bytes(16, d) * (not whole) - 16) / (128 * (d + 2) * 4)
        assert states == 512 * max(1, -(-b * (hq // hkv) // 128) * hkv // 512), (b, keys, whole)


# Sequences, own keys, prefixes, their keys, and whether one launch has both; measured as OWN_KEYS.
JOINED = [
    (32, 8, 128, False, [(2, 300, 1, 16000, True), (4, 300, 1, 8000, True), (16, 300, 1, 1000, True), (16, 300, 1, 2000, False),
                         (16, 1344, 1, 2000, True), (32, 300, 1, 1000, False), (32, 1344, 1, 1000, True), (8, 300, 1, 8000, False),
                         (64, 300, 4, 1000, False)]),
    (32, 8, 128, True, [(16, 300, 1, 2000, True), (32, 300, 1, 2000, False), (48, 1344, 1, 600, True)]),
    (14, 2, 64, False, [(4, 60, 1, 1000, True), (64, 60, 1, 4000, False), (64, 1344, 1, 4000, True), (64, 300, 4, 1000, True)]),
    (8, 8, 64, False, [(64, 300, 1, 1000, False), (32, 300, 1, 2000, False), (16, 1344, 1, 4000, True), (4, 300, 4, 8000, True)]),
]


@pytest.mark.parametrize("hq,hkv,d,q8,sizes", JOINED)
def test_prefix_one_launch_or_two(lib, hq, hkv, d, q8, sizes):
    """One launch has prefixes and own keys where that was measured to be faster."""
    for b, keys, count, prefix_keys, one in sizes:
        p, x = prefix_call(hq, hkv, d, q8, b, keys, prefix_keys, count, page=64 if keys % 64 == 0 else 16)
        size = lib.fa_sm75_paged_prefix_workspace_size(ctypes.byref(p), ctypes.byref(x))
        cut = cut_bytes(16, d)
        assert size == cut if one else size not in (0, cut), (b, keys, count, prefix_keys)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(tokens=-1), 1, b"tokens must be non-negative"),
    (dict(tokens=1), 1, b"a token for each of the 2 sequences"),
    (dict(heads_q=5), 3, b"not divisible"),
    (dict(scale=math.nan), 1, b"finite"),
    (dict(causal=1), 1, b"causal must be 0 or 2"),
    (dict(dtype=-1), 1, b"dtype must be"),
    (dict(q=0), 1, b"Q must not be NULL"),
    (dict(q=0x10008), 4, b"Q must be 16-byte aligned"),
    (dict(q_stride_h=12), 4, b"multiples of 8"),
    (dict(q_stride_h=1 << 23), 5, b"below 2^23"),
    (dict(q_stride_t=1 << 40), 5, b"below 2^23"),
    (dict(heads_q=1 << 10, q_stride_h=1 << 21), 5, b"within 2^30"),
    (dict(lse=0), 1, b"lse must not be NULL"),
    (dict(lse=0x1002), 4, b"lse must be 4-byte aligned"),
    (dict(weights=0), 1, b"weights must not be NULL"),
    (dict(weights=0x1001), 4, b"weights must be 4-byte aligned"),
    (dict(weights_stride_h=-1), 1, b"non-negative"),
    (dict(max_len=-1), 1, b"non-negative"),
    (dict(max_len=(1 << 30) + 1), 5, b"max_len exceeds 2^30"),
    (dict(max_query_len=-1), 1, b"non-negative"),
    (dict(workspace=0x1004, workspace_bytes=64), 4, b"workspace must be 16-byte aligned"),
    (dict(workspace_bytes=-1), 1, b"non-negative"),
])
def test_weigh_refusals(lib, kw, status, msg):
    p = weigh(cache(), **kw)
    assert lib.fa_sm75_paged_weigh(ctypes.byref(p)) == status
    assert msg in lib.fa_sm75_last_error()
    before = lib.fa_sm75_last_error()
    assert lib.fa_sm75_paged_weigh_workspace_size(ctypes.byref(p)) == 0
    assert lib.fa_sm75_last_error() == before


def test_weigh_sizes(lib):
    assert lib.fa_sm75_paged_weigh(None) == 1
    p = weigh(cache())
    p.cache = None
    assert lib.fa_sm75_paged_weigh(ctypes.byref(p)) == 1
    for kw, pk in ((dict(batch=0), dict(tokens=0)), ({}, dict(max_len=0)), ({}, dict(tokens=0, cu_seqlens=0x1000, add=1)),
                   ({}, dict(heads_q=0, add=1))):
        assert lib.fa_sm75_paged_weigh(ctypes.byref(weigh(cache(**kw), **pk))) == 0
    many = weigh(cache(batch=1 << 13, heads_kv=1 << 10), heads_q=0, tokens=1 << 13)
    assert lib.fa_sm75_paged_weigh(ctypes.byref(many)) == 5
    long = weigh(cache(batch=1 << 5), heads_q=0, tokens=1 << 5, max_len=1 << 30)
    assert lib.fa_sm75_paged_weigh(ctypes.byref(long)) == 5
    size = lambda **kw: lib.fa_sm75_paged_weigh_workspace_size(ctypes.byref(weigh(cache(), **kw)))  # noqa: E731
    assert size() == 0  # one row block: never cut
    assert size(cu_seqlens=0x1000, tokens=64) > 0 and size(cu_seqlens=0x1000, tokens=64) % 16 == 0
    assert size(cu_seqlens=0x1000, tokens=64, max_query_len=16) == 0
    # V may be missing
    assert lib.fa_sm75_paged_weigh(ctypes.byref(weigh(cache(v=0, v_stride_n=3, k_scale=0x1000), max_len=0))) == 0


@pytest.mark.parametrize("kw,status,msg", [
    (dict(keep=-1), 1, b"non-negative"),
    (dict(recent=-1), 1, b"non-negative"),
    (dict(to_pages=-1), 1, b"non-negative"),
    (dict(workspace_bytes=-1), 1, b"non-negative"),
    (dict(recent=21), 1, b"recent (21) must not exceed keep (20)"),
    (dict(weights_stride_b=-1), 1, b"non-negative"),
    (dict(to_table_stride=-1), 1, b"non-negative"),
    (dict(to_pages=1 << 40), 5, b"2^30 tokens"),
    (dict(to_pages=1), 1, b"room for 16 rows, up to 20 stay"),
    (dict(keep=1 << 40), 1, b"room for 32 rows, up to 64 stay"),
    (dict(weights_len=63), 1, b"64 positions, got 63"),
    (dict(weights=0), 1, b"must not be NULL"),
    (dict(to_table=0), 1, b"must not be NULL"),
    (dict(new_lens=0), 1, b"must not be NULL"),
    (dict(new_weights=0), 1, b"must not be NULL"),
    (dict(new_lens=0x1002), 4, b"4-byte aligned"),
    (dict(workspace=0), 1, b"must hold 320 bytes, got 0"),
    (dict(workspace_bytes=319), 1, b"must hold 320 bytes, got 319"),
    (dict(workspace=0x1004), 4, b"workspace must be 16-byte aligned"),
])
def test_evict_refusals(lib, kw, status, msg):
    p = evict(cache(), **kw)
    assert lib.fa_sm75_paged_evict(ctypes.byref(p)) == status
    assert msg in lib.fa_sm75_last_error()


def test_evict_in_place_is_refused(lib):
    """Lengths and weights are read while others are written: neither may be the same memory, in part or whole."""
    far = dict(new_lens=0x40000, weights=0x50000, new_weights=0x60000)
    for kw, msg in ((dict(far, new_lens=0x1000), b"new_lens must not share"),
                    (dict(far, new_lens=0x1004), b"new_lens must not share"),
                    (dict(far, new_weights=0x50000), b"new_weights must not share"),
                    (dict(far, new_weights=0x50000 + 4 * 255), b"new_weights must not share"),
                    (dict(far, new_weights=0x50000 - 4 * (2 * 2 * 32 - 1)), b"new_weights must not share")):
        p = evict(cache(), **kw)
        assert p.cache.contents.seq_lens == 0x1000 and p.weights_stride_b == 128
        assert lib.fa_sm75_paged_evict(ctypes.byref(p)) == 1
        assert msg in lib.fa_sm75_last_error()


def test_evict_workspace_of_many_long_rows(lib):
    """The positions of those that stay, and nothing for each digit of each row."""
    size = lambda c, **kw: lib.fa_sm75_paged_evict_workspace_size(ctypes.byref(evict(c, **kw)))  # noqa: E731
    assert size(cache(batch=65, max_pages=1024), weights_len=1 << 14) == 65 * 2 * 20 * 4
    assert size(cache(batch=1 << 18, max_pages=1 << 16), weights_len=1 << 20) == (1 << 18) * 2 * 20 * 4


def test_evict_sizes(lib):
    assert lib.fa_sm75_paged_evict(None) == 1
    assert lib.fa_sm75_paged_evict(ctypes.byref(evict(cache(heads_kv=0)))) == 1
    assert lib.fa_sm75_paged_evict(ctypes.byref(evict(cache(batch=0), new_lens=0))) == 0
    size = lambda c, **kw: lib.fa_sm75_paged_evict_workspace_size(ctypes.byref(evict(c, **kw)))  # noqa: E731
    assert size(cache()) >= 2 * 2 * 20 * 4 and size(cache()) % 16 == 0
    assert size(cache(), keep=10 ** 12, to_pages=4) == size(cache(), keep=64, to_pages=4)  # what there is room for
    assert size(cache(), keep=-1) == 0 and size(cache(batch=0)) == 0
    assert lib.fa_sm75_paged_evict(ctypes.byref(evict(cache(batch=1 << 11, heads_kv=1 << 10)))) == 5


def test_cpu_tensors_and_gradients_are_refused():
    import flash_attention_sm75 as fa
    import torch.autograd.forward_ad as fwd

    c = Cache([5], 2, 64, 16, torch.float16, False)
    (k, v, table, lens), _ = c.args("cpu")
    x, lse, w = torch.zeros(1, 2, 64, dtype=torch.float16), torch.zeros(2, 1), torch.zeros(1, 2, 16)
    calls = {
        "prefix": lambda x=x, k=k, v=v, **kw: fa.flash_attention_paged_prefix(x, k, v, table, lens, table, lens, **kw),
        "weigh": lambda x=x, lse=lse, k=k, **kw: fa.paged_attention_weights(x, lse, k, table, lens, **kw),
        "evict": lambda k=k, v=v, w=w: fa.paged_cache_evict(k, v, table, lens, w, table, 5),
    }
    for call in calls.values():
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    tries = [("prefix", dict(x=leaf(x))), ("prefix", dict(k=leaf(k))), ("prefix", dict(v=leaf(v))),
             ("prefix", dict(out=leaf(x))), ("weigh", dict(x=leaf(x))), ("weigh", dict(lse=leaf(lse))),
             ("weigh", dict(k=leaf(k))), ("weigh", dict(add_to=leaf(w))), ("evict", dict(k=leaf(k))),
             ("evict", dict(v=leaf(v))), ("evict", dict(w=leaf(w)))]
    for name, kw in tries:
        with pytest.raises(RuntimeError, match="no backward pass"):
            calls[name](**kw)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            calls[name](**kw)
    with fwd.dual_level(), torch.no_grad():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for name, kw in tries:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                calls[name](**{n: dual(t.detach()) for n, t in kw.items()})
    for causal in (True, None, "top_left", 2):
        for name in ("prefix", "weigh"):
            with pytest.raises(ValueError, match="bottom_right"):
                calls[name](causal=causal)
    for kw in (dict(max_query_len=-1), dict(max_prefix_queries=-1)):
        with pytest.raises(ValueError, match="non-negative"):
            calls["prefix"](**kw)


# ---- the references --------------------------------------------------------------------


def test_joined_reference_is_attention_over_one_longer_sequence():
    """A prefix that fills its pages is the same as the own table with those pages in front."""
    own, shared = Cache([23, 9], 2, 64, 16, torch.float16, False, news=[5, 12]), Cache([32], 2, 64, 16, torch.float16, False, seed=3)
    q = torch.randn(17, 4, 64).half()
    o, lse, _, _ = ref.attention(con.Joined(own, shared, [0, None]), q)
    k = torch.cat([shared.rows[0][0], own.rows[0][0]], 1).repeat_interleave(2, 0)
    v = torch.cat([shared.rows[0][1], own.rows[0][1]], 1).repeat_interleave(2, 0)
    mask = torch.arange(55)[None] <= torch.arange(50, 55)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q[:5].double().transpose(0, 1)[None], k[None], v[None],
                                                            attn_mask=mask)[0].transpose(0, 1)
    torch.testing.assert_close(o[:5], want, rtol=1e-12, atol=1e-12)
    plain, plain_lse, _, _ = ref.attention(own, q)  # the sequence without a prefix; three tokens see no key
    torch.testing.assert_close(o[5:], plain[5:], rtol=1e-12, atol=1e-12)
    assert (o[5:8] == 0).all() and (lse[:, 5:8] == -math.inf).all()


def test_weights_reference_sums_probabilities():
    c = Cache([40, 7], 2, 64, 16, torch.bfloat16, True, news=[3, 9])
    q = torch.randn(12, 4, 64).bfloat16()
    _, lse, _, _ = ref.attention(c, q)
    w, tol = con.weights(c, q, lse)
    assert abs(float(w[0].sum()) - 12) < 1e-9 and abs(float(w[1].sum()) - 28) < 1e-9  # 2 of 9 tokens see nothing
    assert (tol[w > 0] < 1e-3 * w[w > 0]).all()
    planted = w.clone()
    planted[0, 1, 3] += 2 * tol[0, 1, 3]
    with pytest.raises(AssertionError):
        ref.check(planted, w, tol, "weights")


def test_eviction_reference():
    w = [3.0, math.nan, 1.0, 3.0, 0.0, -0.0, 2.0, 9.0]
    assert con.stays(w, [True] * 8, 8, 3, 0) == [0, 3, 7]
    assert con.stays(w, [True] * 8, 8, 4, 2) == [0, 3, 6, 7]
    assert con.stays(w, [True] * 4 + [False] * 4, 8, 3, 2) == [0, 2, 3]
    assert con.stays(w, [True] * 8, 8, 7, 0) == [0, 2, 3, 4, 5, 6, 7]
    assert con.stays(w, [True] * 8, 8, 5, 0) == [0, 2, 3, 6, 7]
    assert con.stays(w, [True] * 8, 8, 6, 0) == [0, 2, 3, 4, 6, 7]
    assert con.stays(w, [True] * 8, 20, 2, 2) == [0, 7]
