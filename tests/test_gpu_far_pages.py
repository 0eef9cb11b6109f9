"""A cache of more than 4 GiB a side: pages and slots whose byte and element
offsets pass 32 bits, through the in-cache copies, the rotated write and the
shared-prefix decode. Only the pages in use are ever written."""
import ctypes

import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from test_gpu_capi import call, u64

pytestmark = pytest.mark.gpu

HEADS, HD, BS, PAGES = 8, 128, 16, 140_000  # 4.6 GB of K and of V


@pytest.fixture(scope="module")
def cache(cuda):
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of device memory")
    k, v = (torch.empty(PAGES, HEADS, BS, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    desc = kv.KvfxCache(k.data_ptr(), v.data_ptr(), PAGES, HEADS, BS, HD, kv.KVFX_BF16, 0, 0)
    kv.device_status(0, clear=True)
    yield k, v, desc
    del k, v
    torch.cuda.empty_cache()


def test_copies_at_the_far_end(cache):
    k, v, desc = cache
    src, dst = [PAGES - 1, 5, PAGES - 2], [3, PAGES - 3, PAGES - 4]
    for x in (k, v):
        x[src + dst] = torch.randn(6, HEADS, BS, HD, device="cuda").bfloat16()
    want = [x[src].clone() for x in (k, v)]
    call(kv.lib.kvfx_copy_pages, ctypes.byref(desc), 1, u64(src), u64(dst), 3, None)
    for x, w in zip((k, v), want):
        assert torch.equal(x[dst], w)
    s, d = np.array([PAGES * BS - 1, 5 * BS]), np.array([7 * BS + 2, (PAGES - 9) * BS + 11])
    want = [x[s // BS, :, s % BS].clone() for x in (k, v)]
    call(kv.lib.kvfx_copy_slots, ctypes.byref(desc), 1, u64(s), u64(d), 2, None)
    for x, w in zip((k, v), want):
        assert torch.equal(x[d // BS, :, d % BS], w)
    assert kv.device_status(0) == 0


def test_rotated_write_at_the_far_end(cache):
    k, v, desc = cache
    hq = 4
    qkv = torch.randn(3, (hq + 2 * HEADS) * HD, device="cuda").bfloat16()
    table = torch.cat([torch.ones(2, HD // 2), torch.zeros(2, HD // 2)], 1).cuda()  # no turn
    out = torch.zeros(3, hq, HD, device="cuda")
    rotary = kv.KvfxRotary(table.data_ptr(), 2, HD, 0, None, None, 0.0, 0)
    slots = np.array([PAGES * BS - 1, (PAGES - 20) * BS, 40])
    p, w = qkv.data_ptr(), qkv.shape[1]
    call(kv.lib.kvfx_write_rotated, ctypes.byref(desc), ctypes.byref(rotary), p, p + 2 * hq * HD, p + 2 * (hq + HEADS) * HD, w, w, w, hq,
         u64([0, 1, 1]), u64(slots), 3, out, None)
    rows = qkv.view(3, -1, HD)
    assert torch.equal(out, rows[:, :hq].float())
    assert torch.equal(k[slots // BS, :, slots % BS], rows[:, hq:hq + HEADS])
    assert torch.equal(v[slots // BS, :, slots % BS], rows[:, hq + HEADS:])
    assert kv.device_status(0) == 0


def test_shared_decode_over_far_pages(cache):
    """The same contents in near and in far pages give the same bits."""
    k, v, desc = cache
    prefix, rows, own = 50, 6, 3
    n = prefix + rows * own
    near = np.random.default_rng(1).permutation(n) + 100
    far = PAGES - 1 - np.random.default_rng(2).permutation(n)
    for x in (k, v):
        x[near] = torch.randn(n, HEADS, BS, HD, device="cuda").bfloat16()
        x[far] = x[near]
    hq = 16
    q = torch.randn(rows, hq, HD, device="cuda")
    lens = u64([prefix * BS + 1 + 9 * i for i in range(rows)])
    groups = (kv.KvfxPrefixGroup * 1)((rows, prefix * BS))
    need = kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(desc), groups, 1, hq, (prefix + own) * BS)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    got = []
    for ids in (near, far):
        table = np.concatenate([np.tile(ids[:prefix], (rows, 1)), ids[prefix:].reshape(rows, own)], 1)
        o = torch.zeros(rows, hq, HD, device="cuda")
        call(kv.lib.kvfx_decode_shared, ctypes.byref(desc), q, o, u64(table), lens, groups, 1, prefix + own, hq, (prefix + own) * BS, ws, need, None)
        got.append(o)
    assert torch.equal(*got) and torch.isfinite(got[0]).all() and bool((got[0] != 0).all())
    assert kv.device_status(0) == 0


def test_misaligned_cache_runs_row_by_row(cuda):
    """Bases two bytes off a 16-byte boundary: no tensor loads, the same attention."""
    n = 60 * 2 * BS * 64
    buf = torch.randn(2 * n + 1, device="cuda").half()
    out, tables = [], u64(np.concatenate([np.tile(np.arange(50), (2, 1)), [[50], [51]]], 1))
    lens, q = u64([801, 816]), torch.randn(2, 4, 64, device="cuda")
    for shift in (0, 1):
        base = buf.data_ptr() + 2 * shift
        if shift:
            buf[1:] = buf[:-1].clone()
        desc = kv.KvfxCache(base, base + 2 * n, 60, 2, BS, 64, kv.KVFX_F16, 0, 0)
        groups = (kv.KvfxPrefixGroup * 1)((2, 800))
        need = kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(desc), groups, 1, 4, 816)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        o = torch.zeros(2, 4, 64, device="cuda")
        call(kv.lib.kvfx_decode_shared, ctypes.byref(desc), q, o, tables, lens, groups, 1, 51, 4, 816, ws, need, None)
        out.append(o)
    assert float((out[0] - out[1]).abs().max()) < 1e-4 and kv.device_status(0) == 0
