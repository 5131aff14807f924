"""The C entries of the paged cache on the GPU: workspaces of every size, and what they leave alone."""
import ctypes

import pytest
import torch

import paged_ref as ref
from paged_ref import Cache
from test_paged_cpu import PagedCache, PagedParams, lib  # noqa: F401

pytestmark = pytest.mark.gpu


def describe(c, device):
    (k, v, table, lens), kw = c.args(device)
    p = PagedCache(k=k.data_ptr(), v=v.data_ptr(), block_table=table.data_ptr(), seq_lens=lens.data_ptr(),
                   batch=len(c.lens), heads_kv=c.hkv, head_dim=c.d, num_pages=k.shape[0], page_size=c.page,
                   max_pages=table.shape[1], block_table_stride=table.stride(0))
    if kw:
        p.k_scale, p.v_scale = (kw[n].data_ptr() for n in ("k_scale", "v_scale"))
    for n, x, s in (("k", k, kw.get("k_scale")), ("v", v, kw.get("v_scale"))):
        for i, dim in enumerate("phn"):
            setattr(p, f"{n}_stride_{dim}", x.stride(i))
            setattr(p, f"{n}s_stride_{dim}", s.stride(i) if s is not None else 0)
    return p, (k, v, table, lens, kw)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("news,most", [([1, 1, 1], 1), ([4, 1, 2], 4), ([70, 1, 130], 130)])
def test_workspaces(device, lib, news, most, q8):  # noqa: F811
    """Any workspace, none included, gives a right result, and nothing past it is written."""
    c = Cache([3000, 17, 1200], 2, 64, 16, torch.bfloat16, q8, news=news)
    desc, keep = describe(c, device)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(sum(news), 8, 64, generator=g).bfloat16()
    want, want_lse, tol, lse_tol = ref.attention(c, q)
    qd, cu = q.to(device), c.cu.to(device)
    full = None
    for share in (1.0, 0.0, 0.3, 1e-3, 0.011, 2.0):
        o = torch.full_like(qd, 9.0)
        lse = torch.full((8, sum(news)), 9.0, device=device)
        p = PagedParams(cache=ctypes.pointer(desc), q=qd.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(),
                        tokens=sum(news), heads_q=8, q_stride_t=qd.stride(0), q_stride_h=qd.stride(1),
                        o_stride_t=o.stride(0), o_stride_h=o.stride(1), cu_seqlens=cu.data_ptr(),
                        max_query_len=most, scale=0.125, causal=2, dtype=1,
                        stream=torch.cuda.current_stream().cuda_stream)
        full = full or lib.fa_sm75_paged_workspace_size(ctypes.byref(p))
        assert full > 0
        size = int(full * share) // 16 * 16
        room = torch.full((size + 4096,), 77, dtype=torch.uint8, device=device)
        if size:
            p.workspace, p.workspace_bytes = room.data_ptr(), size
        assert lib.fa_sm75_paged_forward(ctypes.byref(p)) == 0
        torch.cuda.synchronize()
        ref.check(o, want, tol, f"O with {size} bytes")
        ref.check(lse, want_lse, lse_tol, f"LSE with {size} bytes")
        assert (room[size:] == 77).all()
    del keep
