"""Paged attention whose units are cut into many pieces: that every row is merged and written, on
either side of where the merge kernel takes over, and that the device cuts as the plan says."""
import ctypes
import os
import random

import pytest
import torch

import flash_attention_sm75 as fa
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


def left(call):
    """Units whose partials the merge kernel takes."""
    plan, _ = call.plan(plans.probe())
    assert plan["split"] and not plan["chunk"]
    return call.left(plan, call.cuts(plan))


MERGED_BY_THE_KERNEL = [
    # (units of a class's line that are left to it, call)
    (1, Call(8, 4, 128, 64, [20000], [4])),
    (1, Call(2, 4, 128, 16, [20011], [4], q8=True)),
    (1, Call(2, 16, 128, 16, [9001], [2])),                                # 32 rows a unit
    (1, Call(2, 16, 128, 32, [9001], [2], q8=True)),
    (1, Call(1, 8, 64, 16, [20001], [4])),
    (1, Call(1, 32, 64, 16, [20001], [1], cu=False, q8=True)),
    (1, Call(1, 16, 128, 64, [12345], [1], cu=False)),
    (3, Call(3, 7, 128, 16, [15001], [4])),                                # three heads of one class
    (2, Call(1, 4, 128, 16, [9000, 30, 12000, 700], [4, 1, 4, 0])),        # unequal ones
    (2, Call(1, 4, 128, 64, [9000, 30, 12000, 700], [4, 4, 4, 4], q8=True)),
    (2, Call(2, 8, 128, 32, [10000, 9500], [3, 4])),
    (4, Call(2, 8, 128, 16, [16384, 16384], [4, 4], hint=1)),              # max_query_len below the truth:
    (3, Call(1, 3, 128, 16, [12000, 50], [15, 1], hint=5)),                # a short last block among them
    (1, Call(2, 4, 128, 16, [20000] + [5] * 70, [4] + [1] * 70)),          # more sequences than lanes
    (1, Call(2, 4, 128, 16, [5] * 70 + [20000], [1] * 70 + [4], q8=True)),
]


@pytest.mark.parametrize("units,call", MERGED_BY_THE_KERNEL, ids=str)
def test_merged_by_the_kernel(device, lib, units, call):  # noqa: F811
    assert len(left(call)) == units
    for dtype in (BF16, FP16):
        o, lse = attend(call, device, lib, dtype)
        again = attend(call, device, lib, dtype)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


def test_merged_by_the_kernel_full_attention(device, lib):  # noqa: F811
    attend(Call(1, 4, 128, 16, [9000, 30, 12000], [4, 1, 4]), device, lib, causal=False)


def test_captured(device):
    """A captured call whose units are left to the merge kernel at some replays and not at others,
    with eager calls of both kinds between them."""
    longest, short = [12000, 40, 9000], [900, 40, 33]
    call = Call(1, 4, 128, 16, longest, [4, 1, 4])
    assert left(call) and not left(Call(1, 4, 128, 16, short, [4, 1, 4], width=call.width))
    c = Cache(longest, 1, 128, 16, BF16, False, news=call.news)
    (k, v, table, lens), _ = c.args(device)
    cu = c.cu.to(device)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(9, 4, 128, generator=g).to(BF16).to(device)

    def attention():
        return fa.flash_attention_paged(q, k, v, table, lens, cu_seqlens=cu, max_query_len=4, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = attention()
    for now in (longest, short, short, longest, longest, short):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g))
        o.fill_(float("nan"))
        lse.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want = attention()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1]), now
        one = Cache(now, 1, 128, 16, BF16, False, news=call.news)
        one.rows = [[x[:, :n] for x in kv] for kv, n in zip(c.rows, now)]
        exact, exact_lse, tol, lse_tol = ref.attention(one, q.cpu())
        ref.check(o, exact, tol, "O")
        ref.check(lse, exact_lse, lse_tol, "LSE")


def test_sweep(device, lib):  # noqa: F811
    """Seeded batches of long sequences and few new tokens, on tables just wide enough and wider,
    to both sides of both decisions: the host's (is the merge kernel launched) and the device's (is
    a unit left to it)."""
    probe, r, seen = plans.probe(), random.Random(21), set()
    todo = int(os.environ.get("FA_PAGED_MERGE_CASES", "60"))
    while todo:
        call = plans.draw(r)
        plan, _ = call.plan(probe)
        if plan["chunk"] or sum(call.lens) * call.hkv * call.d > 1 << 22:
            continue  # (the reference's time)
        seen.add((plan["combine"], bool(plan["split"] and call.left(plan, call.cuts(plan)))))
        attend(call, device, lib, r.choice([FP16, BF16]), causal=r.random() < 0.8)
        todo -= 1
    assert seen >= {(0, False), (1, False), (1, True)}
