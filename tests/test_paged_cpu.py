"""The paged cache without a GPU: refusals of the C ABI and of the Python calls, and the reference itself."""
import ctypes
import math

import pytest
import torch

import paged_ref as ref
from capi_types import LIB
from paged_ref import Cache

I64, PTR, INT = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int


class PagedCache(ctypes.Structure):
    """fa_paged_cache."""
    _fields_ = [(n, PTR) for n in ("k", "v", "k_scale", "v_scale", "block_table", "seq_lens")] + [
        (n, I64) for n in ("batch", "heads_kv", "head_dim", "num_pages", "page_size", "max_pages",
                           "block_table_stride")] + [
        (f"{t}_stride_{d}", I64) for t in ("k", "v", "ks", "vs") for d in "phn"]


class PagedRows(ctypes.Structure):
    """fa_paged_rows."""
    _fields_ = [("k", PTR), ("v", PTR), ("tokens", I64)] + [
        (f"{t}_stride_{d}", I64) for t in "kv" for d in "th"] + [
        ("cu_seqlens", PTR), ("dtype", INT), ("stream", PTR)]


class PagedParams(ctypes.Structure):
    """fa_paged_params."""
    _fields_ = [("cache", ctypes.POINTER(PagedCache)), ("q", PTR), ("o", PTR), ("lse", PTR),
                ("tokens", I64), ("heads_q", I64)] + [
        (f"{t}_stride_{d}", I64) for t in "qo" for d in "th"] + [
        ("cu_seqlens", PTR), ("max_query_len", I64), ("scale", ctypes.c_float), ("causal", INT),
        ("dtype", INT), ("stream", PTR), ("workspace", PTR), ("workspace_bytes", I64)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.fa_sm75_last_error.restype = ctypes.c_char_p
    lib.fa_sm75_paged_write.argtypes = [ctypes.POINTER(PagedCache), ctypes.POINTER(PagedRows)]
    lib.fa_sm75_paged_read.argtypes = [ctypes.POINTER(PagedCache), PTR, PTR, I64, INT, PTR]
    lib.fa_sm75_paged_forward.argtypes = [ctypes.POINTER(PagedParams)]
    lib.fa_sm75_paged_workspace_size.argtypes = [ctypes.POINTER(PagedParams)]
    lib.fa_sm75_paged_workspace_size.restype = I64
    return lib


def cache(**kw):
    c = PagedCache(k=0x10000, v=0x10000, block_table=0x1000, seq_lens=0x1000, batch=2, heads_kv=2,
                   head_dim=64, num_pages=8, page_size=16, max_pages=4, block_table_stride=4)
    for t in "kv":
        for n, x in (("p", 2 * 16 * 64), ("h", 16 * 64), ("n", 64)):
            setattr(c, f"{t}_stride_{n}", x)
        for n, x in (("p", 2 * 16), ("h", 16), ("n", 1)):
            setattr(c, f"{t}s_stride_{n}", x)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rows(**kw):
    r = PagedRows(k=0x10000, v=0x10000, tokens=0, k_stride_t=128, k_stride_h=64, v_stride_t=128,
                  v_stride_h=64, cu_seqlens=0x1000)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def params(c, **kw):
    p = PagedParams(cache=ctypes.pointer(c), q=0x10000, o=0x20000, tokens=2, heads_q=4, q_stride_t=256,
                    q_stride_h=64, o_stride_t=256, o_stride_h=64, scale=0.125, causal=2)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


BAD_CACHES = [
    (dict(head_dim=96), 2, b"head_dim=64 or 128, got 96"),
    (dict(batch=-1), 1, b"non-negative"),
    (dict(max_pages=-1), 1, b"non-negative"),
    (dict(page_size=8), 1, b"power of two from 16"),
    (dict(page_size=48), 1, b"power of two from 16"),
    (dict(page_size=0), 1, b"power of two from 16"),
    (dict(page_size=1 << 21), 1, b"power of two from 16"),
    (dict(batch=1 << 21), 5, b"supported maximum"),
    (dict(num_pages=1 << 31), 5, b"supported maximum"),
    (dict(max_pages=(1 << 26) + 1), 5, b"2^30 tokens"),
    (dict(k_scale=0x1000), 1, b"go together"),
    (dict(seq_lens=0), 1, b"must not be NULL"),
    (dict(block_table=0), 1, b"must not be NULL"),
    (dict(k=0), 1, b"must not be NULL"),
    (dict(v=0x10008), 4, b"16-byte aligned"),
    (dict(seq_lens=0x1002), 4, b"4-byte aligned"),
    (dict(block_table_stride=-4), 1, b"non-negative"),
    (dict(k_stride_h=-64), 1, b"non-negative"),
    (dict(v_stride_n=68), 4, b"multiples of 16 bytes"),
    (dict(k_scale=0x1000, v_scale=0x1000, k_stride_n=72), 4, b"multiples of 16 bytes"),
    (dict(k_stride_n=32), 1, b"at least head_dim"),
    (dict(v_stride_n=1 << 23 | 64), 5, b"2^24 bytes"),
    (dict(k_scale=0x1000, v_scale=0x1000, ks_stride_n=0), 1, b"at least 1"),
    (dict(k_scale=0x1000, v_scale=0x1000, vs_stride_h=-1), 1, b"non-negative"),
]


@pytest.mark.parametrize("kw,status,msg", BAD_CACHES)
def test_cache_refusals(lib, kw, status, msg):
    c = cache(**kw)
    for call in (lambda: lib.fa_sm75_paged_write(ctypes.byref(c), ctypes.byref(rows())),
                 lambda: lib.fa_sm75_paged_read(ctypes.byref(c), 0x10000, 0x10000, 0, 0, None),
                 lambda: lib.fa_sm75_paged_forward(ctypes.byref(params(c)))):
        assert call() == status
        assert msg in lib.fa_sm75_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(tokens=-1), 1, b"tokens must be non-negative"),
    (dict(tokens=(1 << 24) + 1), 5, b"tokens exceeds"),
    (dict(tokens=1, cu_seqlens=0), 1, b"a token for each of the 2 sequences"),
    (dict(tokens=2, cu_seqlens=0x1001), 4, b"4-byte aligned"),
    (dict(tokens=2, dtype=2), 1, b"dtype must be"),
    (dict(tokens=2, k=0), 1, b"K must not be NULL"),
    (dict(tokens=2, v=0x10004), 4, b"V must be 16-byte aligned"),
    (dict(tokens=2, v_stride_t=100), 4, b"multiples of 8"),
    (dict(tokens=2, k_stride_h=-8), 1, b"non-negative"),
])
def test_write_refusals(lib, kw, status, msg):
    assert lib.fa_sm75_paged_write(ctypes.byref(cache()), ctypes.byref(rows(**kw))) == status
    assert msg in lib.fa_sm75_last_error()


def test_write_nulls_and_empty_calls(lib):
    assert lib.fa_sm75_paged_write(None, ctypes.byref(rows())) == 1
    assert lib.fa_sm75_paged_write(ctypes.byref(cache()), None) == 1
    assert lib.fa_sm75_paged_write(ctypes.byref(cache()), ctypes.byref(rows())) == 0
    for kw in (dict(batch=0), dict(heads_kv=0), dict(num_pages=0), dict(max_pages=0)):
        assert lib.fa_sm75_paged_write(ctypes.byref(cache(**kw)), ctypes.byref(rows(tokens=2))) == 0


@pytest.mark.parametrize("args,status,msg", [
    ((0x10000, 0x10000, -1, 0), 1, b"max_len must be non-negative"),
    ((0x10000, 0x10000, 1 << 27, 0), 5, b"2^27 rows"),
    ((0, 0x10000, 16, 0), 1, b"must not be NULL"),
    ((0x10000, 0x10008, 16, 0), 4, b"16-byte aligned"),
    ((0x10000, 0x10000, 16, 5), 1, b"dtype must be"),
])
def test_read_refusals(lib, args, status, msg):
    assert lib.fa_sm75_paged_read(ctypes.byref(cache()), *args, None) == status
    assert msg in lib.fa_sm75_last_error()


def test_read_takes_any_number_of_heads_and_sequences(lib):
    """Only the rows in all are limited (the call ends at the pointer it is not given)."""
    for kw, max_len in ((dict(batch=1024, heads_kv=64), 16), (dict(batch=1 << 20, heads_kv=128), 1)):
        assert lib.fa_sm75_paged_read(ctypes.byref(cache(**kw)), 0, 0x10000, max_len, 0, None) == 1
        assert b"must not be NULL" in lib.fa_sm75_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(tokens=-1), 1, b"tokens must be non-negative"),
    (dict(tokens=1), 1, b"a token for each of the 2 sequences"),
    (dict(heads_q=-2), 1, b"non-negative"),
    (dict(heads_q=5), 3, b"not divisible"),
    (dict(heads_q=1 << 21), 5, b"heads_q exceeds"),
    (dict(scale=math.inf), 1, b"finite"),
    (dict(scale=math.nan), 1, b"finite"),
    (dict(causal=1), 1, b"causal must be 0 or 2"),
    (dict(dtype=-1), 1, b"dtype must be"),
    (dict(q=0), 1, b"Q must not be NULL"),
    (dict(o=0x20008), 4, b"O must be 16-byte aligned"),
    (dict(q_stride_t=12), 4, b"multiples of 8"),
    (dict(o_stride_h=-64), 1, b"non-negative"),
    (dict(lse=0x1002), 4, b"lse must be 4-byte aligned"),
    (dict(workspace=0x1004, workspace_bytes=64), 4, b"workspace must be 16-byte aligned"),
    (dict(workspace_bytes=-1), 1, b"non-negative"),
    (dict(max_query_len=-1), 1, b"non-negative"),
    (dict(tokens=1 << 24, heads_q=16, cu_seqlens=0x1000), 5, b"exceeds 2^27"),
])
def test_forward_refusals(lib, kw, status, msg):
    p = params(cache(), **kw)
    assert lib.fa_sm75_paged_forward(ctypes.byref(p)) == status
    assert msg in lib.fa_sm75_last_error()
    before = lib.fa_sm75_last_error()
    assert lib.fa_sm75_paged_workspace_size(ctypes.byref(p)) == 0  # and no error of its own
    assert lib.fa_sm75_last_error() == before


def test_forward_nulls_and_empty_calls(lib):
    assert lib.fa_sm75_paged_forward(None) == 1
    p = params(cache())
    p.cache = None
    assert lib.fa_sm75_paged_forward(ctypes.byref(p)) == 1
    for kw, pk in ((dict(batch=0), dict(tokens=0)), ({}, dict(tokens=0, cu_seqlens=0x1000)), ({}, dict(heads_q=0))):
        p = params(cache(**kw), q=0, o=0, **pk)
        assert lib.fa_sm75_paged_forward(ctypes.byref(p)) == 0
        assert lib.fa_sm75_paged_workspace_size(ctypes.byref(p)) == 0
    assert lib.fa_sm75_paged_forward(ctypes.byref(params(cache(heads_kv=0)))) == 3


def test_workspace_sizes(lib):
    """Of the sizes alone, whole 16 bytes, none for a call that cannot split."""
    c = cache(batch=4, heads_kv=8, head_dim=128, max_pages=512, block_table_stride=512,
              **{f"{t}_stride_n": 128 for t in "kv"})
    size = lambda **kw: lib.fa_sm75_paged_workspace_size(ctypes.byref(params(c, heads_q=32, **kw)))  # noqa: E731
    one = size(tokens=4)
    assert one > 0 and one % 16 == 0
    few, chunk = size(tokens=16, cu_seqlens=0x1000, max_query_len=4), size(tokens=256, cu_seqlens=0x1000)
    assert few > 0 and few % 16 == 0 and chunk > 0 and chunk % 16 == 0
    assert size(tokens=256, cu_seqlens=0x1000, max_query_len=2 ** 63 - 1) == chunk
    assert size(tokens=1 << 20, cu_seqlens=0x1000) == 0  # a workgroup for each block fills the GPU


# ---- the Python calls ------------------------------------------------------------


def test_cpu_tensors_are_refused():
    import flash_attention_sm75 as fa

    c = Cache([5], 2, 64, 16, torch.float16, False)
    args, _ = c.args("cpu")
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.flash_attention_paged(x, *args)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.paged_cache_write(x, x, *args)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.paged_cache_read(*args)


def test_python_refusals():
    import flash_attention_sm75 as fa

    c = Cache([5], 2, 64, 16, torch.float16, False)
    args, _ = c.args("cpu")
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    for causal in (True, "top_left", None, 2):
        with pytest.raises(ValueError, match="bottom_right"):
            fa.flash_attention_paged(x, *args, causal=causal)
    with pytest.raises(ValueError, match="max_query_len"):
        fa.flash_attention_paged(x, *args, max_query_len=-1)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        fa.flash_attention_paged(leaf, *args)
    with pytest.raises(RuntimeError, match="no backward pass"):
        fa.paged_cache_write(leaf, x, *args)
    with pytest.raises(RuntimeError, match="no backward pass"):
        fa.flash_attention_paged(x, *args, out=leaf)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):  # past that check
        fa.flash_attention_paged(leaf, *args)


def test_tangents_are_refused():
    """Forward-mode derivatives are not computed, so an input that carries one is not taken for a
    plain tensor; with forward mode off, and of the primals, the calls go on (to the next check)."""
    import flash_attention_sm75 as fa
    import torch.autograd.forward_ad as fwd

    c = Cache([5], 2, 64, 16, torch.float16, False)
    (k, v, table, lens), _ = c.args("cpu")
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    calls = [lambda y, kc, vc: fa.paged_cache_write(y, x, kc, vc, table, lens),
             lambda y, kc, vc: fa.paged_cache_write(x, y, kc, vc, table, lens),
             lambda y, kc, vc: fa.flash_attention_paged(y, kc, vc, table, lens),
             lambda y, kc, vc: fa.flash_attention_paged(x, kc, vc, table, lens, out=y)]
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        pool = fwd.make_dual(k, torch.ones_like(k))
        with torch.no_grad():
            for call in calls:
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(dual, k, v)
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(x, pool, v)
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(x, v, pool)
                with pytest.raises(RuntimeError, match="CUDA"):
                    call(fwd.unpack_dual(dual).primal, k, v)
            for args in ((pool, v), (v, pool)):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    fa.paged_cache_read(*args, table, lens)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="CUDA"):
            fa.flash_attention_paged(dual, k, v, table, lens)


# ---- the reference ------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantiser(dtype):
    """The scale is the smallest power of two with max |x| <= 448 s, codes are within half a step,
    and what they stand for is a number of the 16-bit type."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(2000, 64, generator=g) * torch.exp2(torch.randint(-16, 12, (2000, 1), generator=g).float())).to(dtype)
    codes, scale = ref.quantise(x)
    s, amax = scale.double(), x.double().abs().amax(-1)
    assert (amax <= 448 * s).all()
    assert ((amax > 224 * s) | (s == 2.0 ** -126)).all()
    y = codes.double() * s[:, None]
    err = (y - x.double()).abs()
    assert (err <= torch.maximum(x.double().abs() * 2.0 ** -4, s[:, None] * 2.0 ** -10)).all()
    assert torch.equal(y.to(dtype).double(), y)


def test_reference_matches_dense_attention():
    """With nothing missing, the paged reference is causal attention of the last tokens."""
    c = Cache([40, 23], 2, 64, 16, torch.float16, False, news=[7, 23])
    q = torch.randn(30, 4, 64).half()
    o, lse, tol, _ = ref.attention(c, q)
    for b in range(2):
        n, L, t0 = c.news[b], c.lens[b], int(c.cu[b])
        k, v = (x.repeat_interleave(2, 0) for x in c.rows[b])
        mask = torch.arange(L)[None] <= torch.arange(L - n, L)[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(q[t0:t0 + n].double().transpose(0, 1)[None], k[None],
                                                                v[None], attn_mask=mask)[0].transpose(0, 1)
        torch.testing.assert_close(o[t0:t0 + n], want, rtol=1e-12, atol=1e-12)
    planted = o.clone()
    planted[5, 1, 3] += 2 * tol[5, 1, 3]
    with pytest.raises(AssertionError):
        ref.check(planted, o, tol, "O")
