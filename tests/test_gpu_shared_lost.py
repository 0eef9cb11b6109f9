"""kvfx_decode_shared when its prefix kernel gives up: the rows behind a prefix
are NaN and not a join with the pieces that an earlier call left in the
workspace; the others are untouched by it."""
import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from test_gpu_capi import call, u64
from test_gpu_shared_decode import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,lens,heads,group,hd,dtype", [
    ([(4, 800), (3, 0)], [800, 816, 1000, 1056, 5, 700, 33], 2, 4, 128, "bfloat16"),       # tails that join the pieces
    ([(3, 320), (2, 0)], [320, 336, 6000, 17, 5000], 2, 9, 64, "float16"),                 # the merge kernel
    ([(50, 1040), (1, 0), (2, 640)], [1040 + i for i in range(50)] + [600, 640, 700], 3, 4, 128, "float16"),
    ([(9, 128 * 37)], [128 * 37] * 9, 1, 7, 128, "bfloat16"),                              # no row has pages of its own
])
def test_lost_pieces_are_not_taken_from_an_earlier_call(cuda, groups, lens, heads, group, hd, dtype):
    kv.device_status(0, clear=True)
    b = Batch(groups, lens, heads, group, hd, dtype=dtype)
    b.check(b.run())  # leaves its pieces in the workspace
    out = torch.full((len(lens), b.hq, hd), 7.0, device="cuda")
    call(kv.lib.kvfx_selftest_lost_prefix, *b.args(out))
    got = out.cpu()
    prefixes = [p for n, p in groups for _ in range(n)]
    behind = [r for r, p in enumerate(prefixes) if p]
    assert torch.all(torch.isnan(got[behind]))
    b.check(got, rows=[r for r, p in enumerate(prefixes) if not p])
    b.check(b.run())
    assert kv.device_status(0) == 0


def test_calls_without_a_prefix_kernel_lose_nothing(cuda):
    b = Batch([(3, 64)], [64, 80, 100], 2, 4, 128)  # one launch reads the shared pages too
    out = torch.full((3, b.hq, 128), 7.0, device="cuda")
    call(kv.lib.kvfx_selftest_lost_prefix, *b.args(out))
    b.check(out.cpu())
    b = Batch([(2, 800)], [810, 820], 2, 4, 128)
    b.dlens = u64(np.array([0, 2000], np.uint64))  # padding and a refused row stay as they were
    out = torch.full((2, b.hq, 128), 7.0, device="cuda")
    call(kv.lib.kvfx_selftest_lost_prefix, *b.args(out))
    assert torch.all(out == 7.0)
    assert kv.device_status(0, clear=True) == kv.KVFX_FLAG_BAD_INDEX
