"""kvfx_copy_pages and kvfx_copy_slots: byte-exact against the same copies of a
host mirror, over every vector width (rows of 16-byte multiples down to odd
element counts), several layers, repeated sources, single copies, the last
page and slot of a pool, out-of-range ids, and graph replay on a side stream.
Bytes that no copy names stay as they were."""
import ctypes

import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from kvflux_b200 import workloads as w
from test_gpu_capi import Cache, call, u64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clear_status(cuda):
    kv.device_status(0, clear=True)
    yield


SHAPES = [  # dtype, head_size, block_size, kv_heads, layers
    ("bfloat16", 128, 16, 8, 3),
    ("float16", 64, 16, 2, 1),
    ("float32", 32, 8, 3, 2),
    ("bfloat16", 12, 16, 2, 2),   # 24-byte rows: 8-byte vectors
    ("float32", 3, 6, 2, 2),      # 12-byte rows, block size no power of two
    ("bfloat16", 5, 7, 3, 2),     # 10-byte rows
    ("float16", 1, 1, 1, 1),      # one element a page
]


def layers_of(n, nb, heads, bs, hd, dtype, seed):
    caches = [Cache(nb, heads, bs, hd, dtype, seed=seed + 17 * i) for i in range(n)]
    return caches, (kv.KvfxCache * n)(*[c.desc for c in caches])


def pages_view(raw, c):
    return raw.reshape(c.nb, c.h, c.bs, c.row)


def expect(caches, move):
    for c in caches:
        for raw in (c.host_k, c.host_v):
            move(pages_view(raw, c))
        gk, gv = c.device_bytes()
        assert np.array_equal(gk, c.host_k) and np.array_equal(gv, c.host_v)


@pytest.mark.parametrize("dtype,hd,bs,heads,layers", SHAPES)
@pytest.mark.parametrize("n,fan", [(1, 1), (7, 1), (16, 5)])
def test_copy_pages(dtype, hd, bs, heads, layers, n, fan):
    nb = 41
    caches, arr = layers_of(layers, nb, heads, bs, hd, dtype, seed=3)
    ids = w.permutation(n + hd, np.arange(nb))
    src, dst = np.repeat(ids[:-(-n // fan)], fan)[:n], ids[nb - n:]
    call(kv.lib.kvfx_copy_pages, arr, layers, u64(src), u64(dst), n, None)

    def move(pages):
        pages[dst] = pages[src]

    expect(caches, move)
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("dtype,hd,bs,heads,layers", SHAPES)
@pytest.mark.parametrize("n", [1, 15, 16, 33])
def test_copy_slots(dtype, hd, bs, heads, layers, n):
    nb = max(41, -(-80 // bs))
    caches, arr = layers_of(layers, nb, heads, bs, hd, dtype, seed=5)
    slots = w.permutation(n + hd, np.arange(nb * bs))
    src, dst = np.sort(slots[:n]), slots[nb * bs - n:]
    src[0], dst[-1] = slots[n], slots[n + 1]
    call(kv.lib.kvfx_copy_slots, arr, layers, u64(src), u64(dst), n, None)

    def move(pages):
        rows = pages.transpose(0, 2, 1, 3)
        rows[dst // bs, dst % bs] = rows[src // bs, src % bs]

    expect(caches, move)
    assert kv.device_status(0) == 0


def test_unaligned_bases_and_the_last_page():
    """A cache that starts two bytes off a 16-byte boundary; first to last page."""
    nb, heads, bs, hd = 5, 2, 4, 8
    n = nb * heads * bs * hd
    host = w.encode(w.normal(9, 2 * n + 1), "bfloat16")
    buf = torch.from_numpy(host.view(np.int16).copy()).cuda()
    base = buf.data_ptr() + 2
    desc = kv.KvfxCache(base, base + 2 * n, nb, heads, bs, hd, kv.KVFX_BF16, 0, 0)
    call(kv.lib.kvfx_copy_pages, ctypes.byref(desc), 1, u64([0]), u64([nb - 1]), 1, None)
    want = host.copy()
    per = heads * bs * hd
    for first in (1, 1 + n):
        want[first + (nb - 1) * per:first + nb * per] = want[first:first + per]
    assert np.array_equal(buf.cpu().numpy().view(np.uint16), want)


@pytest.mark.parametrize("fn,limit", [("kvfx_copy_pages", 12), ("kvfx_copy_slots", 12 * 16)])
def test_bad_ids_are_skipped_and_flagged(fn, limit):
    caches, arr = layers_of(2, 12, 2, 16, 64, "bfloat16", seed=7)
    src = np.array([0, limit, 2, 3, 2**64 - 1], np.uint64)
    dst = np.array([5, 6, limit, 8, 9], np.uint64)
    call(getattr(kv.lib, fn), arr, 2, u64(src), u64(dst), 5, None)
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX

    def move(pages):
        if fn == "kvfx_copy_pages":
            pages[[5, 8]] = pages[[0, 3]]
        else:
            pages[0, :, [5, 8]] = pages[0, :, [0, 3]]

    expect(caches, move)


def test_replayed_graph_reads_the_ids_of_the_day():
    caches, arr = layers_of(2, 40, 2, 16, 64, "float16", seed=11)
    src, dst = u64([1, 2, 3]), u64([20, 21, 22])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        kv.check(kv.lib.kvfx_copy_pages(arr, 2, src.data_ptr(), dst.data_ptr(), 3, side.cuda_stream), "capture")
    src.copy_(u64([4, 5, 4]))
    dst.copy_(u64([30, 39, 31]))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()

    def move(pages):
        pages[[30, 39, 31]] = pages[[4, 5, 4]]

    expect(caches, move)
