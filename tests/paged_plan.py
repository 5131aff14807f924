"""How an attention call over a paged cache is cut, for the tests of it: the host's plan from
the library, and the device's whole-number arithmetic (PagedLine, PagedStretch, PagedPieces and
paged_stretch of fa_paged_units.h and fa_paged_attn.h) written again.
"""
import ctypes
import math
import os

import pytest

PROBE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "probe", "libpaged_plan.so")
TILE, LEAST, AHEAD = 32, 8, 3  # kPTile, kPMinTiles, kPAhead
MERGE_BYTES, THREADS = 256 << 10, 256  # kPMergeBytes, kThreads


def probe():
    if not os.path.exists(PROBE):
        pytest.fail(f"{PROBE} not built: run __graft_entry__.build()")
    lib = ctypes.CDLL(PROBE)
    lib.fa_probe_paged_plan.restype = None
    lib.fa_probe_paged_plan.argtypes = [ctypes.c_int] * 9 + [ctypes.c_int64] * 2 + [ctypes.c_void_p]
    lib.fa_probe_paged_pieces.argtypes = ([ctypes.c_int] * 7 + [ctypes.c_void_p] * 4 + [ctypes.c_int])
    return lib


class Call:
    """lens and news: tokens and new tokens of each sequence; width: pages of the table."""

    def __init__(self, hkv, group, d, page, lens, news, width=None, cu=True, q8=False, hint=None,
                 workspace=2 ** 62):
        self.hkv, self.group, self.d, self.page, self.lens, self.news = hkv, group, d, page, lens, news
        self.width = max(-(-n // page) for n in lens) if width is None else width
        self.cu, self.q8, self.workspace = cu, q8, workspace
        self.hint = (max(news) if hint is None else hint) if cu else 1

    def __repr__(self):
        def short(x):
            return str(x) if len(x) <= 16 else f"{len(x)} from {x[0]} to {x[-1]}"
        return (f"{self.hkv * self.group} over {self.hkv} heads d{self.d} page {self.page} lens {short(self.lens)} "
                f"news {short(self.news)} width {self.width} cu {self.cu} q8 {self.q8} max_query_len {self.hint}")

    def sizes(self):
        return (self.hkv, self.group, len(self.lens), sum(self.news), self.d, self.page.bit_length() - 1, self.width)

    def plan(self, lib):
        got = (ctypes.c_int * 7)()
        lib.fa_probe_paged_plan(*self.sizes(), int(self.cu), int(self.q8), self.hint, self.workspace, got)
        names = ("classes", "wgs", "rows", "split", "combine", "chunk", "pieces")
        return dict(zip(names, got)), got

    def unit_rows(self, rows):
        """Rows of every unit of a class, in the order of its line."""
        heads = self.hkv // math.gcd(self.hkv, 8)
        got = []
        for n in self.news:
            r = n * self.group
            got += [min(rows, r - i) for i in range(0, r, rows)] * heads
        return got

    def cuts(self, plan):
        """Pieces of every unit of a class (the kernel for few columns)."""
        rows, heads, wgs = plan["rows"], self.hkv // plan["classes"], plan["wgs"]
        tiles = [-(-min(n, self.width * self.page) // TILE) for n in self.lens]
        blocks = [-(-n * self.group // rows) for n in self.news]
        looked = {t for t, n in zip(tiles[:64], self.news[:64]) if n > 0}
        ahead = AHEAD if len(looked) > 1 else 0
        same = max(1, *looked, 1) if len(looked) <= 1 and len(tiles) <= 64 else 0
        total = heads * sum(b * (ahead + max(1, t)) for b, t in zip(blocks, tiles))
        active = cuts = min(wgs, -(-total // LEAST))
        length = total
        if same and active:
            count = max(1, total // same)
            q = min(wgs // count, -(-same // LEAST))
            if q > 0 and same <= q * (total // active + AHEAD):
                active, length, cuts = count * q, same, q
        if not active:
            return []
        size, longer = divmod(length, cuts)

        def holder(pos):
            u, x = divmod(pos, length)
            p = x - longer * (size + 1)
            return u * cuts + (x // (size + 1) if p < 0 else longer + p // size)

        got, at = [], 0
        for b, t in zip(blocks, tiles):
            for _ in range(heads * b):
                end = at + ahead + max(1, t)
                got.append(holder(end - 1) - holder(at + ahead) + 1)
                at = end
        return got

    def left(self, plan, pieces):
        """Units that are left to the merge kernel: (index, pieces, rows)."""
        if plan["chunk"]:
            most = (320 << 10) // (128 * self.d * 4)  # chunk_pieces
            return [(i, p, 128) for i, p in enumerate(pieces) if p > most]
        rows = self.unit_rows(plan["rows"])
        return [(i, p, r) for i, (p, r) in enumerate(zip(pieces, rows))
                if p > 1 and (p > THREADS or p * r * self.d * 4 > MERGE_BYTES)]


# Batches whose longest unit is cut into as many pieces as the bound on them allows: one more
# than the last workgroup merges.
AT_THE_BOUND = [
    Call(8, 8, 128, 16, [32, 3744, 64], [4, 4, 4]),
    Call(8, 4, 128, 16, [32, 7883, 268], [4, 4, 4]),
    Call(1, 16, 128, 16, [25, 7896, 3], [1, 1, 1], cu=False),
    Call(1, 8, 128, 16, [28, 15974, 95], [1, 1, 1], cu=False),
    Call(8, 1, 128, 64, [7453, 7835, 126, 94], [16, 16, 16, 16]),
    Call(8, 4, 128, 32, [20, 3800, 20], [1, 8, 1]),
    Call(8, 4, 128, 32, [20, 7900, 20], [1, 4, 1]),
    Call(2, 8, 64, 16, [20, 7900, 20], [1, 4, 1]),
]


def draw(r):
    """A batch of few new tokens; every second one with a sequence about as long as a unit is whose
    partials the last workgroup just merges."""
    d = r.choice([64, 128])
    hkv = r.choice([1, 1, 2, 3, 8, 16])
    group = r.choice([1, 4, 7, 8, 16, 32])
    rows = r.choice([16, 32])
    n = max(1, rows // group) if r.random() < 0.8 else r.randint(1, max(1, 32 // group))
    b = r.choice([1, 2, 3, 3, 4, 6, 12])
    lens = [int(math.exp(r.uniform(0, math.log(r.choice([100, 3000, 9000]))))) for _ in range(b)]
    if r.random() < 0.5:
        most = MERGE_BYTES // (min(rows, n * group) * d * 4)
        lens[r.randrange(b)] = max(n, TILE * LEAST * (most - 2) + r.randint(-TILE, TILE * LEAST + TILE))
    news = [n if r.random() < 0.7 else r.randint(0, n) for _ in lens]
    if not any(news):
        news[0] = n
    page = r.choice([16, 16, 32, 64, 256])
    cu = not (n == 1 and all(x == 1 for x in news)) or r.random() < 0.5
    width = None if r.random() < 0.7 else -(-max(lens) // page) + r.choice([0, 1, 2, 7, 100])
    hint = None if r.random() < 0.8 else r.choice([1, 2, 4])
    return Call(hkv, group, d, page, lens, news, width, cu, r.random() < 0.5, hint)
