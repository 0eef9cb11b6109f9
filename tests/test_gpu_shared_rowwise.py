"""kvfx_decode_shared on the shapes it takes row by row (FP32, other head or
block sizes, misaligned bases): the same contract as on the others. Batch and
its tolerance are those of test_gpu_shared_decode."""
import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from test_gpu_capi import u64
from test_gpu_shared_decode import Batch

pytestmark = pytest.mark.gpu

# dtype, hd, bs, the base that is not on 16 bytes
SHAPES = [("float32", 32, 8, None), ("float32", 128, 16, None), ("bfloat16", 80, 16, None), ("float16", 64, 32, None),
          ("bfloat16", 128, 16, "cache"), ("float16", 64, 16, "q")]


@pytest.fixture(autouse=True)
def clear_status(cuda):
    kv.device_status(0, clear=True)
    yield


def shifted(t):
    """The same values one element past a 16-byte boundary."""
    room = torch.empty(t.numel() + 16 // t.element_size(), dtype=t.dtype, device="cuda")
    out = room[1:1 + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 != 0
    return out


def batch(shape, groups, lens, **kw):
    dtype, hd, bs, odd = shape
    b = Batch(groups, lens, 2, 4, hd, bs, dtype, **kw)
    if odd == "cache":
        b.dk = shifted(b.dk)
        b.cache.k_base = b.dk.data_ptr()
    elif odd == "q":
        b.dq = shifted(b.dq)
    return b


@pytest.mark.parametrize("room", [0, 1000])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_outside_their_bounds_are_refused(shape, room):
    """Shorter than the prefix, or above max_seq_len (where the table row still has pages): untouched and flagged."""
    b = batch(shape, [(4, 256)], [256, 300, 400, 290], room=room)
    b.dlens = u64(np.array([255, 300, 401 + room, 240], np.uint64))
    got = b.run()
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    b.check(got, rows=[1])
    assert torch.all(got[[0, 2, 3]] == 7.0)
    kv.device_status(0, clear=True)
    b.dlens = u64(np.array([256, 2**63, 0, 290], np.uint64))
    got = b.run()
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    b.check(got, rows=[0, 3])
    assert torch.all(got[1:3] == 7.0)


@pytest.mark.parametrize("shape", SHAPES)
def test_every_group_has_its_own_bound(shape):
    groups, lens = [(2, 64), (1, 0), (2, 320)], [64, 100, 5, 320, 333]
    b = batch(shape, groups, lens)
    b.check(b.run())
    assert kv.device_status(0) == 0
    b.dlens = u64(np.array([63, 100, 1, 319, 333], np.uint64))
    got = b.run()
    assert kv.device_status(0) == kv.KVFX_FLAG_BAD_INDEX
    b.check(got, lens=[64, 100, 1, 320, 333], rows=[1, 2, 4])
    assert torch.all(got[[0, 3]] == 7.0)


@pytest.mark.parametrize("first", [300, 0])
@pytest.mark.parametrize("shape", SHAPES)
def test_only_the_first_row_names_the_prefix(shape, first):
    """The other rows' entries for it are not read; the first row's are, also where that row is padding."""
    lens = [first, 270, 256, 70, 64]
    b = batch(shape, [(3, 256), (2, 64)], lens)
    table = b.table.copy()
    table[1:3, : 256 // b.bs] = b.pages + 5
    table[4, : 64 // b.bs] = b.pages + 5
    b.dtable = u64(table)
    b.check(b.run())
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("tokens", [32, 256])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] != "float16"])  # fp16 holds no such keys
def test_scores_below_the_lowest_value_weigh_nothing(shape, tokens):
    """-2e38 x 4 a dimension sums past FP32's range: such a score is -inf, its weight 0, wherever it stands."""
    b = batch(shape, [(3, 256)], [300, 270, 257])
    b.q.fill_(4.0)
    b.dq.copy_(b.q)
    b.poison(-2e38, [int(x) for x in b.table[0, : tokens // b.bs]])
    b.check(b.run())
    assert kv.device_status(0) == 0


@pytest.mark.parametrize("shape", SHAPES)
def test_scores_of_nan_come_through(shape):
    b = batch(shape, [(3, 256)], [300, 270, 257])
    b.poison(float("nan"), [int(x) for x in b.table[0, : 32 // b.bs]], 0)  # the first 32 scores, in one of two heads
    got = b.run().view(3, 2, 4, b.hd)
    assert torch.all(torch.isnan(got[:, 0])) and torch.all(torch.isfinite(got[:, 1]))
    assert kv.device_status(0) == 0
