"""kvfx_decode_shared against the attention of every row in 64 bits through
the row's own table: groups of one to many rows, prefixes of no, one and many
pages that end inside a 128-token tile, query tiles that are full, partial and
several, query groups above 8 heads, rows with no tokens of their own, padding
rows, refused rows, bad pages, large scores, shapes without a fast kernel,
graph replay and two calls in flight.

Tolerance, per output. Q and the softmax weights are pairs of 16-bit values:
each is off by at most 2^-17 of itself (bf16, of x in [1, 2): the high part's unit
is 2^-7, so the low part is at most 2^-8, with a unit of 2^-16 of which half is lost; fp16's 2^-22 has a floor of 2^-25
for weights whose low part is below its smallest step). With A = the largest
sum |q_i k_i| / sqrt(hd) of the row, a score is off by at most
A (2^-17 + hd 2^-23), counting one truncation of an FP32 accumulator an
addend; that is each weight's relative error, and the sum's, so it counts
twice. Weights add 2^-17 and 2^-21 for the exponential and the joins, the
accumulation of n addends n 2^-23. All count against W = sum p |v|."""
import ctypes
import math

import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from test_gpu_capi import call, u64

pytestmark = pytest.mark.gpu

TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


@pytest.fixture(autouse=True)
def clear_status(cuda):
    kv.device_status(0, clear=True)
    yield


class Batch:
    """Rows on a permuted pool whose unwritten slots hold NaN."""

    def __init__(self, groups, lens, heads, group, hd, bs=16, dtype="bfloat16", seed=1, q_scale=1.0, k_drift=0.0, room=0):
        self.groups, self.lens, self.heads, self.hq, self.hd, self.bs, self.dtype = groups, lens, heads, heads * group, hd, bs, dtype
        gen = torch.Generator().manual_seed(seed)
        rows = [g for g, (n, _) in enumerate(groups) for _ in range(n)]
        assert len(rows) == len(lens)
        # `room`: the host's bound above the longest row. Past 640 tokens the groups' prefixes are shared by the
        # tensor-core kernel; below, one launch reads row by row (as long as the rows fit one wave).
        self.max_len = max(max(lens), max(p for _, p in groups)) + room
        self.width = -(-self.max_len // bs) + 2
        self.table = np.full((len(rows), self.width), 2**64 - 1, np.uint64)
        need = sum(p // bs for _, p in groups) + sum(max(0, -(-n // bs) - groups[g][1] // bs) for g, n in zip(rows, lens))
        ids = iter(torch.randperm(need + 3, generator=gen).tolist())
        self.pages = need + 3
        shared = [[next(ids) for _ in range(p // bs)] for _, p in groups]
        self.k = torch.full((self.pages, heads, bs, hd), float("nan"), dtype=TORCH[dtype])
        self.v = self.k.clone()
        for r, (g, n) in enumerate(zip(rows, lens)):
            pre = groups[g][1] // bs
            self.table[r, :pre] = shared[g]
            for j in range(pre, -(-n // bs)):
                self.table[r, j] = next(ids)
        written = set()
        for r, (g, n) in enumerate(zip(rows, lens)):
            for j in range(max(-(-n // bs), groups[g][1] // bs)):
                page = int(self.table[r, j])
                if page in written:
                    continue
                written.add(page)
                live = bs if j < groups[g][1] // bs else min(bs, n - j * bs)
                for c in (self.k, self.v):
                    c[page, :, :live] = torch.randn(heads, live, hd, generator=gen).to(TORCH[dtype])
                if k_drift:  # later positions score higher: the running maximum keeps moving
                    self.k[page, :, :live] += (k_drift * j)
        self.q = q_scale * torch.randn(len(rows), self.hq, hd, generator=gen)
        if k_drift:
            self.q = self.q.abs()
        self.dk, self.dv, self.dq = self.k.cuda(), self.v.cuda(), self.q.cuda()
        self.cache = kv.KvfxCache(self.dk.data_ptr(), self.dv.data_ptr(), self.pages, heads, bs, hd, kv.DTYPE_CODE[dtype], 0, 0)
        self.dtable, self.dlens = u64(self.table), u64(np.array(lens, np.uint64))
        self.c_groups = (kv.KvfxPrefixGroup * len(groups))(*groups)
        self.need = kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(self.cache), self.c_groups, len(groups), self.hq, self.max_len)
        # Whatever the workspace held must not matter.
        self.ws = torch.full((max(self.need, 16),), 255, dtype=torch.uint8, device="cuda")

    def args(self, out, stream=None, ws=None):
        ws = self.ws if ws is None else ws
        return (ctypes.byref(self.cache), self.dq.data_ptr(), out.data_ptr(), self.dtable.data_ptr(), self.dlens.data_ptr(), self.c_groups,
                len(self.groups), self.width, self.hq, self.max_len, ws.data_ptr(), self.need, stream)

    def run(self, **kw):
        out = torch.full((len(self.lens), self.hq, self.hd), 7.0, device="cuda")
        call(kv.lib.kvfx_decode_shared, *self.args(out, **kw))
        return out.cpu()

    def check(self, got, lens=None, rows=None, adds=None):
        lens = self.lens if lens is None else lens
        for r, n in enumerate(lens):
            if rows is not None and r not in rows:
                continue
            if n == 0:
                assert torch.all(got[r] == 7.0), r
                continue
            t = np.arange(n)
            page, off = self.table[r, t // self.bs].astype(np.int64), t % self.bs
            k, v = (x[page, :, off].double().permute(1, 0, 2) for x in (self.k, self.v))
            q = self.q[r].double().view(self.heads, -1, self.hd)
            p = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(self.hd), -1)
            want, weight = p @ v, p @ v.abs()
            seen = torch.where(k.abs() > 1e30, 0.0, k.abs())  # (scores past FP32's lowest value weigh exactly 0)
            a = (q.abs() @ seen.transpose(1, 2)).amax(-1, keepdim=True) / math.sqrt(self.hd)
            split = 0.0 if self.dtype == "float32" else 2.0**-17
            tol = weight * (2 * a * (split + self.hd * 2.0**-23) + split + 2.0**-21 + (adds or n) * 2.0**-23)
            if self.dtype == "float16":
                tol = tol + n * 2.0**-25 * v.abs().max()
            err = (got[r].double().view(self.heads, -1, self.hd) - want).abs()
            assert torch.all(err <= tol), (r, n, float((err / tol).max()))


    def poison(self, key, pages, heads=slice(None)):
        self.k[pages, heads] = key
        self.dk.copy_(self.k)


CASES = [  # groups (rows, prefix), lens, heads, q_group, hd, bs, dtype
    ([(4, 512)], [512, 513, 530, 544], 2, 4, 128, 16, "bfloat16"),
    ([(1, 16), (3, 2064), (2, 0), (5, 144)], [17, 2064, 2065, 3000, 1, 400, 144, 145, 160, 161, 500], 2, 4, 64, 16, "float16"),
    ([(2, 16)], [16, 16], 1, 1, 128, 16, "float16"),
    ([(1, 128)], [129], 1, 8, 64, 16, "bfloat16"),
    ([(50, 1040)], [1040 + 7 * i % 90 for i in range(50)], 3, 4, 128, 16, "bfloat16"),        # two query tiles, the second partial
    ([(64, 256)], [256 + i for i in range(64)], 1, 4, 64, 16, "bfloat16"),                     # exactly two query tiles
    ([(3, 48), (2, 320)], [48, 49, 100, 321, 999], 2, 12, 128, 16, "float16"),                 # q_group above 8
    ([(9, 128 * 37)], [128 * 37 + 1] * 9, 1, 7, 128, 16, "bfloat16"),                          # one pair over many CTAs
    ([(2, 16 * (1 + g % 11)) for g in range(32)], [16 * (1 + g // 2 % 11) + g % 5 for g in range(64)], 2, 2, 64, 16, "bfloat16"),
    ([(4, 256), (3, 160)], [0, 256, 300, 0, 0, 0, 0], 2, 4, 128, 16, "bfloat16"),              # padding rows, a group of nothing else
    ([(3, 0)], [1, 33, 700], 2, 4, 128, 16, "bfloat16"),                                       # nothing shared
    ([(3, 64), (2, 0)], [64, 70, 0, 5, 129], 2, 2, 32, 8, "float32"),                          # row by row
    ([(2, 32)], [33, 0], 1, 3, 80, 16, "bfloat16"),
    ([(2, 64)], [90, 64], 2, 16, 64, 32, "float16"),
]


@pytest.mark.parametrize("room", [0, 1000])
@pytest.mark.parametrize("groups,lens,heads,group,hd,bs,dtype", CASES)
def test_against_every_row_alone(groups, lens, heads, group, hd, bs, dtype, room):
    b = Batch(groups, lens, heads, group, hd, bs, dtype, room=room)
    got = b.run()
    assert kv.device_status(0) == 0
    b.check(got)
    assert torch.equal(got, b.run())  # the same bits again


@pytest.mark.parametrize("groups,lens,heads,group,hd", [
    # rows that fill the GPU: one split a row, joined by its own CTA; some with nothing of their own, some refused later
    ([(100, 320), (60, 0), (40, 16)], [320 + 5 * i % 700 if i < 100 else 16 + 11 * i % 900 for i in range(200)], 2, 3, 64),
    # short rows of few: likewise
    ([(5, 800)], [800, 801, 1000, 1056, 816], 1, 8, 128),
    # few rows, long of their own: several splits and the merge kernel
    ([(3, 160)], [6000, 160, 3000], 2, 9, 64),
    # one row's split longer than 64 pages a warp
    ([(300, 32)], [32 + (i % 3) for i in range(299)] + [5200], 1, 1, 64),
])
def test_one_split_a_row_and_several(groups, lens, heads, group, hd):
    b = Batch(groups, lens, heads, group, hd)
    b.check(b.run())
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("dtype,hd", [("bfloat16", 128), ("float16", 64)])
def test_large_and_growing_scores(dtype, hd):
    groups, lens = [(5, 1200)], [1200, 1201, 1300, 1250, 1216]
    b = Batch(groups, lens, 2, 4, hd, dtype=dtype, q_scale=6.0)
    b.check(b.run())
    b = Batch(groups, lens, 2, 4, hd, dtype=dtype, k_drift=0.125)
    b.check(b.run())
    assert kv.device_status(0) == 0


# One launch, row by row; tails that join the prefix's pieces; a merge of several splits.
FORMS = [([(3, 64)], [64, 80, 100], 0), ([(4, 800)], [800, 816, 1000, 1056], 0), ([(3, 320)], [320, 336, 900], 1000)]


@pytest.mark.parametrize("groups,lens,room", FORMS)
def test_scores_of_nan_come_through(groups, lens, room):
    b = Batch(groups, lens, 2, 4, 128, room=room)
    shared = [int(x) for x in b.table[0, : groups[0][1] // 16]]
    b.poison(float("nan"), shared, 0)  # every score of the prefix, in one of two heads
    got = b.run().view(len(lens), 2, 4, 128)
    assert torch.all(torch.isnan(got[:, 0])) and torch.all(torch.isfinite(got[:, 1]))
    b = Batch(groups, lens, 2, 4, 128, room=room)
    b.poison(float("nan"), int(b.table[1, groups[0][1] // 16]), 1)  # the second row's first page of its own
    got = b.run().view(len(lens), 2, 4, 128)
    assert torch.all(torch.isnan(got[1, 1])) and torch.all(torch.isfinite(got[1, 0]))
    assert torch.all(torch.isfinite(got[[0, 2]]))
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("where", ["first page", "prefix", "own pages"])
@pytest.mark.parametrize("groups,lens,room", FORMS)
def test_scores_below_the_lowest_value_weigh_nothing(groups, lens, room, where):
    # -2e38 x 4 a dimension sums past FP32's range: the score is -inf, its weight 0.
    b = Batch(groups, lens, 2, 4, 128, room=room)
    pre = groups[0][1] // 16
    b.q.fill_(4.0)
    b.dq.copy_(b.q)
    rows = range(len(lens))
    if where == "first page":
        pages = [int(b.table[0, 0])]
    elif where == "prefix":
        pages, rows = [int(x) for x in b.table[0, :pre]], [r for r in rows if lens[r] > groups[0][1]]
    else:
        pages = sorted({int(b.table[r, j]) for r in rows for j in range(pre, -(-lens[r] // 16))})
    b.poison(-2e38, pages)
    b.check(b.run(), rows=rows)
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("pages", [1 << 18, 1 << 19])
def test_prefixes_of_more_tiles_than_a_block_joins(pages):
    # A few pages over and over: the attention of those few, which is what it
    # is compared with. A group ahead moves the runs off the prefix's first tile.
    distinct, hd, bs = 64, 64, 16
    b = Batch([(1, 8 * bs), (2, distinct * bs)], [8 * bs, distinct * bs, distinct * bs], 1, 4, hd)
    width = pages + 2
    table = np.zeros((3, width), np.uint64)
    table[0, : pages - 8] = np.tile(b.table[0, :8], pages // 8 - 1)
    table[1:, :pages] = np.tile(b.table[1, :distinct], pages // distinct)
    sizes = [(pages - 8) * bs, pages * bs]
    lens, groups = np.array([sizes[0], sizes[1], sizes[1]], np.uint64), (kv.KvfxPrefixGroup * 2)((1, sizes[0]), (2, sizes[1]))
    reach = pages * bs + 16
    need = kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(b.cache), groups, 2, 4, reach)
    out, ws = torch.full((3, 4, hd), 7.0, device="cuda"), torch.empty(need, dtype=torch.uint8, device="cuda")
    call(kv.lib.kvfx_decode_shared, ctypes.byref(b.cache), b.dq, out, u64(table), u64(lens), groups, 2, width, 4, reach, ws, need, None)
    torch.cuda.synchronize()
    assert kv.device_status(0) == 0
    # One accumulator takes at most 8 tiles of 128 tokens before a sum that rounds takes it: 1024 truncated
    # additions, then half a unit each for a run's 32 of those and the runs' join (at most 258), and for the
    # weights' sum (7 levels within a tile, 256 tiles, the join): 1024 + (32 + 258 + 7 + 256 + 258) / 2.
    b.check(out.cpu(), adds=1430)


@pytest.mark.parametrize("room", [0, 1000])
def test_rows_outside_their_bounds_are_refused(room):
    b = Batch([(4, 256)], [256, 300, 400, 290], 2, 4, 128, room=room)
    lens = [255, 300, 401 + room, 240]
    b.dlens = u64(np.array(lens, np.uint64))
    got = b.run()
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    b.check(got, rows=[1])
    assert torch.all(got[[0, 2, 3]] == 7.0)
    b.dlens = u64(np.array([256, 2**63, 400, 290], np.uint64))
    got = b.run()
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    b.check(got, rows=[0, 2, 3])
    assert torch.all(got[1] == 7.0)


@pytest.mark.parametrize("room", [0, 1000])
@pytest.mark.parametrize("row,col", [(0, 3), (1, 17)])
def test_bad_pages_are_flagged(row, col, room):
    """A prefix page (of the group's first row) or a row's own page outside the pool."""
    b = Batch([(2, 256)], [300, 300], 2, 4, 128, room=room)
    table = b.table.copy()
    table[row, col] = b.pages
    b.dtable = u64(table)
    got = b.run()
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    if row == 1:
        b.check(got, rows=[0])


@pytest.mark.parametrize("room", [0, 1000])
def test_only_the_first_row_names_the_prefix(room):
    b = Batch([(3, 256)], [300, 270, 256], 2, 4, 128, room=room)
    table = b.table.copy()
    table[1:, :16] = b.pages + 5
    b.dtable = u64(table)
    b.check(b.run())
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("room", [0, 1000])
def test_replayed_graph_reads_the_lengths_of_the_day(room):
    b = Batch([(3, 256), (2, 32)], [300, 400, 256, 40, 33], 2, 4, 128, room=room)
    out = torch.full((5, b.hq, b.hd), 7.0, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        kv.check(kv.lib.kvfx_decode_shared(*b.args(out, stream=side.cuda_stream)), "capture")
        kv.check(kv.lib.kvfx_decode_shared(*b.args(out, stream=side.cuda_stream)), "capture")
    for lens in ([300, 400, 256, 40, 33], [257, 0, 256, 32, 0]):
        out.fill_(7.0)
        b.dlens.copy_(u64(np.array(lens, np.uint64)))
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        b.check(out.cpu(), lens=lens)
    assert kv.device_status(0) == 0


def test_two_streams_with_workspaces_of_their_own():
    a = Batch([(20, 1024)], [1024 + i for i in range(20)], 2, 4, 128, seed=2)
    b = Batch([(12, 640), (3, 16)], [700] * 15, 4, 2, 64, dtype="float16", seed=3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.full((len(x.lens), x.hq, x.hd), 7.0, device="cuda") for x in (a, b)]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, o, s in zip((a, b), outs, streams):
            kv.check(kv.lib.kvfx_decode_shared(*x.args(o, stream=s.cuda_stream)), "stream")
    torch.cuda.synchronize()
    a.check(outs[0].cpu())
    b.check(outs[1].cpu())
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("room", [0, 1000])
def test_agrees_with_the_plain_decode(room):
    b = Batch([(6, 512)], [520 + 3 * i for i in range(6)], 2, 4, 128, room=room)
    got = b.run()
    need = kv.lib.kvfx_decode_workspace_bytes(ctypes.byref(b.cache), 6, b.hq, b.max_len, 0)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    out = torch.zeros(6, b.hq, b.hd, device="cuda")
    call(kv.lib.kvfx_decode, ctypes.byref(b.cache), b.dq, out, b.dtable, b.dlens, 6, b.width, b.hq, b.max_len, 0, ws, need, None)
    b.check(out.cpu())
    b.check(got)


def test_captured_forks_beside_an_eager_call():
    """A capture on one stream while another stream's eager call uses a workspace of its own."""
    a = Batch([(4, 1040)], [1040, 1100, 1300, 1041], 2, 4, 64, seed=5)
    b = Batch([(4, 1040)], [1040, 1100, 1300, 1041], 2, 4, 64, seed=6)
    outs = [torch.full((4, 8, 64), 7.0, device="cuda") for _ in range(2)]
    side, other, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        kv.check(kv.lib.kvfx_decode_shared(*a.args(outs[0], stream=side.cuda_stream)), "capture")
    graph.replay()
    kv.check(kv.lib.kvfx_decode_shared(*b.args(outs[1], stream=other.cuda_stream)), "eager")
    graph.replay()
    torch.cuda.synchronize()
    a.check(outs[0].cpu())
    b.check(outs[1].cpu())


def test_lengths_rows_and_heads_at_random():
    """Seeded shapes over the whole range: groups, rows, prefixes, own tokens, heads, types."""
    rng = np.random.default_rng(7)
    for i in range(24):
        heads, group = int(rng.choice([1, 2, 3])), int(rng.choice([1, 2, 3, 5, 8, 12]))
        groups = [(int(rng.integers(1, 40 // (g + 1) + 1)), int(rng.integers(0, 90)) * 16) for g in range(int(rng.integers(1, 5)))]
        lens = [p + int(rng.choice([0, 1, 15, 16, 17, int(rng.integers(1, 400))])) for n, p in groups for _ in range(n)]
        lens = [n if rng.random() > 0.1 else 0 for n in lens]
        if not any(lens):
            lens[0] = groups[0][1] + 1
        b = Batch(groups, lens, heads, group, int(rng.choice([64, 128])), dtype=str(rng.choice(["float16", "bfloat16"])), seed=100 + i,
                  room=int(rng.choice([0, 1000])))
        b.check(b.run())
        assert kv.device_status(0) == 0
