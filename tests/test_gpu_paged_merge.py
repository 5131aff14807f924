"""Paged attention whose units are cut into many pieces: that every row is merged and written, on
either side of where the merge kernel takes over, and that the device cuts as the plan says."""
import ctypes
import random

import pytest
import torch

import paged_plan as plans
import paged_ref as ref
from paged_plan import AT_THE_BOUND, Call
from paged_ref import Cache
from test_gpu_paged_capi import describe
from test_paged_cpu import PagedParams, lib  # noqa: F401

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def attend(call, device, lib, dtype=BF16, causal=True):  # noqa: F811
    """The call through the C entry, on O and LSE full of NaN, against the 64-bit reference;
    returns both."""
    c = Cache(call.lens, call.hkv, call.d, call.page, dtype, call.q8, news=call.news, width=call.width)
    hq, t = call.hkv * call.group, sum(call.news)
    q = torch.randn(t, hq, call.d, generator=torch.Generator().manual_seed(1)).to(dtype)
    desc, keep = describe(c, device)
    qd, cu = q.to(device), c.cu.to(device)
    o = torch.full_like(qd, float("nan"))
    lse = torch.full((hq, t), float("nan"), device=device)
    p = PagedParams(cache=ctypes.pointer(desc), q=qd.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(), tokens=t,
                    heads_q=hq, q_stride_t=qd.stride(0), q_stride_h=qd.stride(1), o_stride_t=o.stride(0),
                    o_stride_h=o.stride(1), cu_seqlens=cu.data_ptr() if call.cu else None,
                    max_query_len=call.hint, scale=call.d ** -0.5, causal=2 if causal else 0,
                    dtype=int(dtype == BF16), stream=torch.cuda.current_stream().cuda_stream)
    size = lib.fa_sm75_paged_workspace_size(ctypes.byref(p))
    room = torch.empty(max(size, 16), dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = room.data_ptr(), size
    print(f"{call} {dtype} causal {causal}", flush=True)
    assert lib.fa_sm75_paged_forward(ctypes.byref(p)) == 0
    torch.cuda.synchronize()
    want, want_lse, tol, lse_tol = ref.attention(c, q, causal)
    ref.check(o, want, tol, "O")
    ref.check(lse, want_lse, lse_tol, "LSE")
    del keep
    return o, lse


@pytest.mark.parametrize("call", AT_THE_BOUND, ids=str)
def test_units_at_the_bound(device, lib, call):  # noqa: F811
    attend(call, device, lib)


def test_the_device_cuts_as_planned(device):
    """Pieces of every unit: the device's own against the arithmetic the CPU tests use (few
    columns), and none past what the host's plan provides for (both kernels)."""
    probe, r = plans.probe(), random.Random(12)
    few = chunk = 0
    while few < 150 or chunk < 50:
        call = plans.draw(r)
        if chunk < 50 and r.random() < 0.4:
            call.hint, call.cu = 10 ** 6, True
        plan, raw = call.plan(probe)
        if not plan["split"]:
            continue
        rows = call.unit_rows(plan["rows"])
        lens = torch.tensor(call.lens, dtype=torch.int32, device=device)
        cu = torch.tensor([0] + call.news, device=device).cumsum(0).int()
        got = torch.zeros(len(rows), dtype=torch.int32, device=device)
        torch.cuda.synchronize()
        assert probe.fa_probe_paged_pieces(*call.sizes(), lens.data_ptr(), cu.data_ptr() if call.cu else None, raw,
                                           got.data_ptr(), len(rows)) == 0
        pieces = got.tolist()
        if not plan["chunk"]:
            assert pieces == call.cuts(plan), call
        left = call.left(plan, pieces)
        assert plan["combine"] or not left, f"{call}: nobody merges units {left}"
        few, chunk = few + (not plan["chunk"]), chunk + plan["chunk"]
