"""Refusals of the in-cache copies, the rotated write and the rotary table
that need no GPU: each returns its code before touching CUDA."""
import ctypes

import kvflux_b200 as kv
from test_capi_cpu import _cache


def test_copies_refuse_bad_arguments():
    two = (kv.KvfxCache * 2)(_cache(), _cache(k_base=16384, v_base=20480))
    odd = (kv.KvfxCache * 2)(_cache(), _cache(head_size=16))
    for f in (kv.lib.kvfx_copy_pages, kv.lib.kvfx_copy_slots):
        assert f(None, 2, 1, 1, 1, None) == kv.KVFX_EINVAL
        assert f(two, kv.KVFX_MAX_LAYERS + 1, 1, 1, 1, None) == kv.KVFX_EINVAL
        assert f(odd, 2, 1, 1, 1, None) == kv.KVFX_EINVAL
        assert f(two, 2, None, 1, 1, None) == kv.KVFX_EINVAL
        assert f(two, 2, 1, None, 1, None) == kv.KVFX_EINVAL
        assert f(two, 2, 1, 1, 4 * 16 + 1, None) == kv.KVFX_EINVAL  # more than the pool's slots
        big = (kv.KvfxCache * 1)(_cache(block_size=2**20, head_size=2**12))
        assert f(big, 1, 1, 1, 1, None) == kv.KVFX_EINVAL            # pages above 1 GiB
        assert f(two, 2, None, None, 0, None) == kv.KVFX_OK
        assert f(two, 0, None, None, 5, None) == kv.KVFX_OK
    assert b"1 GiB" in kv.lib.kvfx_last_error()


def _rotary(**kw):
    d = dict(cos_sin=4096, max_positions=10, rotary_dim=8, interleaved=0, q_weight=None, k_weight=None, eps=1e-6, reserved=0)
    d.update(kw)
    return ctypes.byref(kv.KvfxRotary(**d))


def test_rotated_write_refuses_bad_arguments():
    c = ctypes.byref(_cache())  # 2 heads of 8

    def f(rotary=None, q=1, k=1, v=1, sq=32, sk=16, sv=16, hq=4, pos=1, slots=1, n=1, out=1, cache=c):
        return kv.lib.kvfx_write_rotated(cache, rotary or _rotary(), q, k, v, sq, sk, sv, hq, pos, slots, n, out, None)

    assert kv.lib.kvfx_write_rotated(c, None, 1, 1, 1, 32, 16, 16, 4, 1, 1, 1, 1, None) == kv.KVFX_EINVAL
    assert f(cache=None) == kv.KVFX_EINVAL
    for bad in (dict(cos_sin=None), dict(max_positions=0), dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=10), dict(interleaved=2),
                dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(reserved=1)):
        assert f(_rotary(**bad)) == kv.KVFX_EINVAL, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(out=None), dict(sq=31), dict(sk=15), dict(sv=15),
                dict(hq=2**31)):
        assert f(**bad) == kv.KVFX_EINVAL, bad
    assert f(sk=2**62) == kv.KVFX_EOVERFLOW
    assert f(k=None, v=None, pos=None, slots=None, n=0) == kv.KVFX_OK


def test_rotary_table_refuses_bad_arguments():
    f = kv.lib.kvfx_rotary_table
    assert f(None, 4, 8, 10000.0, 1.0, 0, None) == kv.KVFX_EINVAL
    for reach, rot, base, scale, device in ((0, 8, 1e4, 1.0, 0), (4, 0, 1e4, 1.0, 0), (4, 7, 1e4, 1.0, 0), (4, 8, 0.0, 1.0, 0),
                                            (4, 8, float("nan"), 1.0, 0), (4, 8, 1e4, float("inf"), 0), (4, 8, 1e4, 1.0, -1)):
        assert f(1, reach, rot, base, scale, device, None) == kv.KVFX_EINVAL
    assert f(1, 2**61, 8, 1e4, 1.0, 0, None) == kv.KVFX_EOVERFLOW


def test_shared_decode_refuses_bad_arguments():
    c = ctypes.byref(_cache())  # 2 heads, pages of 16

    def f(groups=((2, 32),), n=None, q=16, o=16, table=16, lens=16, width=4, hq=4, max_len=64, ws=None, ws_bytes=0):
        arr = (kv.KvfxPrefixGroup * max(1, len(groups)))(*groups) if groups is not None else None
        n = len(groups) if n is None else n
        return kv.lib.kvfx_decode_shared(c, q, o, table, lens, arr, n, width, hq, max_len, ws, ws_bytes, None)

    assert kv.lib.kvfx_decode_shared(None, 1, 1, 1, 1, None, 0, 4, 4, 64, None, 0, None) == kv.KVFX_EINVAL
    assert f(groups=(), q=None, o=None, table=None, lens=None) == kv.KVFX_OK
    for bad in (dict(hq=3), dict(hq=0), dict(groups=None, n=1), dict(groups=((0, 32),)), dict(groups=((2, 33),)), dict(groups=((2, 80),)),
                dict(groups=((65535, 0), (1, 0))), dict(groups=((2**63, 0), (2**63, 0))), dict(groups=((1, 0),) * 33), dict(q=None), dict(o=None),
                dict(table=None), dict(lens=None), dict(width=3), dict(max_len=0)):
        assert f(**bad) == kv.KVFX_EINVAL, bad
    fast = _cache(num_blocks=1024, num_kv_heads=8, head_size=128)
    groups = (kv.KvfxPrefixGroup * 2)((8, 512), (3, 0))
    need = kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(fast), groups, 2, 32, 1024)
    assert need > 0
    call = kv.lib.kvfx_decode_shared
    assert call(ctypes.byref(fast), 16, 16, 16, 16, groups, 2, 64, 32, 1024, 256, need - 1, None) == kv.KVFX_ENOSPACE
    assert call(ctypes.byref(fast), 16, 16, 16, 16, groups, 2, 64, 32, 1024, None, need, None) == kv.KVFX_ENOSPACE
    assert call(ctypes.byref(fast), 16, 16, 16, 16, groups, 2, 64, 32, 1024, 264, need, None) == kv.KVFX_EINVAL
    # row-by-row shapes need none; refused arguments size none
    assert kv.lib.kvfx_decode_shared_workspace_bytes(c, groups, 2, 4, 1024) == 0
    assert kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(fast), groups, 2, 30, 1024) == 0
