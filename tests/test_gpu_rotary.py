"""kvfx_rotary_table and kvfx_write_rotated against the same formulas in 64
bits: both pairings, partial rotation, with and without norms, packed and
strided inputs, the vector kernel's head sizes and the element-wise one's,
padding tokens, no Q heads, odd token counts, and far positions.

Tolerances. The FP32 value of a dimension comes from at most hd + 8 roundings
of half a unit each: hd in the sum of squares, whose relative error the square
root halves (rsqrtf itself is within two units, four halves), two for scale
and weight, three for the rotation's products and sum. Each counts against
|a cos| + |b sin| <= |a| + |b|. K adds its type's half unit, and half of FP16's
smallest step."""
import ctypes

import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from test_gpu_capi import Cache, call, u64

pytestmark = pytest.mark.gpu

TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


@pytest.fixture(autouse=True)
def clear_status(cuda):
    kv.device_status(0, clear=True)
    yield


def table64(reach, rot, base=10000.0, scale=1.0):
    angle = np.arange(reach, dtype=np.float64)[:, None] * scale * base ** (-np.arange(0, rot, 2) / rot)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1)


@pytest.mark.parametrize("reach,rot,base,scale", [(1, 2, 10000.0, 1.0), (1000, 128, 10000.0, 1.0), (777, 6, 500000.0, 0.25)])
def test_table(reach, rot, base, scale):
    out = torch.full((reach * rot + 1,), 7.0, device="cuda")
    call(kv.lib.kvfx_rotary_table, out, reach, rot, base, scale, 0, None)
    want = table64(reach, rot, base, scale)
    got = out.cpu().numpy()
    assert got[-1] == 7.0
    # Angles up to reach * scale carry a few FP64 roundings; then one FP32 rounding.
    err = np.abs(got[:-1].reshape(reach, rot) - want)
    assert np.all(err <= np.abs(want) * 2.0**-24 + 2.0**-50 * (reach * scale + 1))


def reference(x, weight, eps, cos, sin, rot, interleaved):
    """(y, bound) in 64 bits: x [n][heads][hd]; bound is |a| + |b| of each dimension's pair."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    size = np.abs(y)
    first = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    a, b = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return y, size


CASES = [  # dtype, hd, bs, q_heads, kv_heads, rot, interleaved, norm, tokens, pad (elements between tokens)
    ("bfloat16", 128, 16, 8, 2, 128, 0, True, 37, 0),
    ("bfloat16", 128, 16, 32, 8, 128, 0, True, 1, 0),
    ("float16", 64, 16, 5, 1, 32, 1, True, 33, 8),
    ("float16", 64, 16, 3, 3, 64, 0, False, 700, 0),
    ("float32", 128, 16, 4, 2, 64, 0, True, 5, 4),
    ("float32", 256, 8, 2, 1, 256, 1, True, 9, 0),
    ("bfloat16", 256, 16, 7, 7, 128, 0, True, 11, 0),
    ("bfloat16", 32, 4, 4, 4, 16, 0, True, 300, 0),
    ("bfloat16", 32, 4, 41, 4, 8, 1, False, 13, 0),
    ("bfloat16", 96, 16, 4, 2, 96, 0, True, 21, 0),      # element-wise: head size
    ("float16", 128, 16, 4, 2, 20, 0, True, 21, 0),      # element-wise: rotary_dim 20
    ("float32", 64, 16, 3, 1, 64, 1, True, 17, 3),       # element-wise: stride not of 16 bytes
    ("bfloat16", 2, 3, 3, 1, 2, 0, True, 19, 1),
    ("float32", 5, 2, 2, 2, 4, 1, False, 8, 0),
    ("bfloat16", 128, 16, 0, 2, 128, 0, True, 15, 0),    # no Q
]


@pytest.mark.parametrize("dtype,hd,bs,hq,hkv,rot,inter,norm,n,pad", CASES)
def test_write_rotated(dtype, hd, bs, hq, hkv, rot, inter, norm, n, pad):
    eps, reach = 1e-5, 5000
    gen = torch.Generator().manual_seed(hd * n + rot)
    nb = -(-n // bs) + 3
    cache = Cache(nb, hkv, bs, hd, dtype, seed=13)
    width = (hq + 2 * hkv) * hd + pad
    qkv = torch.randn(n, width, generator=gen).to(TORCH[dtype])
    if dtype == "float16":
        qkv[0, :] *= 2.0**-14  # a row near the type's smallest values
    table = torch.from_numpy(table64(reach, rot)).float()
    wq, wk = (1 + 0.2 * torch.randn(hd, generator=gen) for _ in range(2))
    pos = torch.randint(0, reach, (n,), generator=gen)
    pos[-1] = reach - 1
    slots = torch.randperm(nb * bs, generator=gen)[:n].numpy().astype(np.uint64)
    padding = n // 3 if n > 3 else None
    if padding is not None:
        slots[padding] = kv.KVFX_NO_SLOT
        pos[padding] = 10**12  # not looked at
    dev, dt, dwq, dwk = qkv.cuda(), table.cuda(), wq.cuda(), wk.cuda()
    out = torch.full((n * hq * hd + 4,), 5.0, device="cuda")
    rotary = kv.KvfxRotary(dt.data_ptr(), reach, rot, inter, dwq.data_ptr() if norm else None, dwk.data_ptr() if norm else None, eps, 0)
    e = dev.element_size()
    q, k, v = (dev.data_ptr() + x * hd * e for x in (0, hq, hq + hkv))
    call(kv.lib.kvfx_write_rotated, ctypes.byref(cache.desc), ctypes.byref(rotary), q if hq else None, k, v, width, width, width, hq,
         u64(pos.numpy().astype(np.uint64)), u64(slots), n, out if hq else None, None)
    assert kv.device_status(0) == 0

    live = np.array([s != kv.KVFX_NO_SLOT for s in slots])
    x = qkv.double().numpy()[:, :(hq + 2 * hkv) * hd].reshape(n, -1, hd)[live]
    rows = table.double().numpy()[pos.numpy()[live]][:, None]
    cos, sin = rows[..., :rot // 2], rows[..., rot // 2:]
    steps = (hd + 8) * 2.0**-24
    got = out.cpu().numpy()
    assert np.all(got[n * hq * hd:] == 5.0)
    got = got[:n * hq * hd].reshape(n, hq, hd)
    assert np.all(got[~live] == 5.0)
    want, size = reference(x[:, :hq], wq.double().numpy() if norm else None, eps, cos, sin, rot, inter)
    assert np.all(np.abs(got[live] - want) <= steps * size)

    want, size = reference(x[:, hq:hq + hkv], wk.double().numpy() if norm else None, eps, cos, sin, rot, inter)
    gk, gv = cache.device_bytes()
    at = slots[live].astype(np.int64)
    half = {"float16": 2.0**-11, "bfloat16": 2.0**-8, "float32": 2.0**-24}[dtype]
    tiny = 2.0**-25 if dtype == "float16" else 0.0

    def rows_of(raw):
        t = torch.from_numpy(raw.copy()).view(TORCH[dtype]).view(nb, hkv, bs, hd)
        return t[at // bs, :, at % bs]

    err = np.abs(rows_of(gk).double().numpy() - want)
    assert np.all(err <= steps * size * (1 + half) + half * np.abs(want) + tiny)
    assert torch.equal(rows_of(gv), qkv[torch.from_numpy(live)][:, (hq + hkv) * hd:(hq + 2 * hkv) * hd].view(-1, hkv, hd))
    # Everything else in the cache is as it was.
    for raw, old in ((gk, cache.host_k), (gv, cache.host_v)):
        r, o = (z.reshape(nb, hkv, bs, cache.row).copy() for z in (raw, old))
        r[at // bs, :, at % bs] = o[at // bs, :, at % bs]
        assert np.array_equal(r, o)


def test_bad_slots_and_positions_are_skipped_and_flagged():
    cache = Cache(4, 2, 16, 64, "bfloat16", seed=17)
    n, hq, reach = 4, 4, 50
    qkv = torch.randn(n, (hq + 4) * 64).bfloat16().cuda()
    table = torch.from_numpy(table64(reach, 64)).float().cuda()
    out = torch.full((n, hq, 64), 5.0, device="cuda")
    rotary = kv.KvfxRotary(table.data_ptr(), reach, 64, 0, None, None, 0.0, 0)
    q = qkv.data_ptr()
    call(kv.lib.kvfx_write_rotated, ctypes.byref(cache.desc), ctypes.byref(rotary), q, q + hq * 128, q + (hq + 2) * 128, 512, 512, 512, hq,
         u64([1, reach, 2, 3]), u64([0, 1, 64, 2**63]), n, out, None)
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    got = out.cpu()
    assert torch.all(got[1:] == 5.0) and not torch.any(got[0] == 5.0)
    gk, gv = cache.device_bytes()
    same = (gk.reshape(4, 2, 16, 128) == cache.host_k.reshape(4, 2, 16, 128)).all(-1)
    same[0, :, 0] = True
    assert same.all()


def test_an_infinity_past_rotary_dim_stays():
    for dtype, inter in (("float16", 0), ("bfloat16", 1), ("float32", 0)):
        c = Cache(4, 1, 16, 128, dtype, seed=23)
        q = torch.randn(3, 2 * 128).to(TORCH[dtype]).cuda()
        k, v = q[:, :128].contiguous(), q[:, 128:].contiguous()
        q[1, 100], k[2, 64], q[0, 127] = float("inf"), float("-inf"), float("inf")
        tab = torch.tensor(table64(8, 64), dtype=torch.float32, device="cuda")
        out = torch.zeros(3, 2, 128, device="cuda")
        rotary = kv.KvfxRotary(tab.data_ptr(), 8, 64, inter, None, None, 0.0, 0)
        call(kv.lib.kvfx_write_rotated, ctypes.byref(c.desc), ctypes.byref(rotary), q, k, v, 256, 128, 128, 2, u64(np.arange(3)), u64(np.arange(3)), 3, out, None)
        assert torch.equal(out[:, :, 64:], q.view(3, 2, 128)[:, :, 64:].float())
        assert torch.all(torch.isfinite(out[:, :, :64]))
        got = torch.from_numpy(c.device_bytes()[0].copy()).view(TORCH[dtype]).view(4, 16, 128)[0, :3, 64:]
        assert torch.equal(got, k[:, 64:].cpu())


def test_rows_of_zeros_and_of_infinities():
    """A zero row norms to zero (eps keeps it finite); an infinite element spoils its own head only."""
    cache = Cache(2, 1, 16, 64, "float16", seed=19)
    hq, reach = 2, 8
    qkv = torch.ones(2, 4 * 64).half()
    qkv[0, :64] = 0
    qkv[1, 70] = float("inf")
    dev = qkv.cuda()
    table = torch.from_numpy(table64(reach, 64)).float().cuda()
    ones = torch.ones(64, device="cuda")
    out = torch.zeros(2, hq, 64, device="cuda")
    rotary = kv.KvfxRotary(table.data_ptr(), reach, 64, 0, ones.data_ptr(), ones.data_ptr(), 1e-6, 0)
    q = dev.data_ptr()
    call(kv.lib.kvfx_write_rotated, ctypes.byref(cache.desc), ctypes.byref(rotary), q, q + hq * 128, q + 3 * 128, 256, 256, 256, hq,
         u64([0, 3]), u64([0, 1]), 2, out, None)
    got = out.cpu()
    assert torch.all(got[0, 0] == 0)
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1, 0]).all()
    assert torch.isnan(got[1, 1, [6, 38]]).all()  # inf / inf, and its rotation partner
