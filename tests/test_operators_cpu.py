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
