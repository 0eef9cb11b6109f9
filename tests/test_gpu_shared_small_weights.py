"""Weights at both ends of fp16's range, in fp16 caches. Small ones: many
tokens of weight near 2^-26 behind one of weight 1 in every page, whose own
value is 0, so that the output is what the small weights carry. Large ones:
scores near 2^26, whose unit is 8, that grow in steps of 8 and 16, with
values of 1, so that the output is 1 whatever the weights are.

Tolerance. A weight is a pair of fp16 values: off by at most 2^-23 of itself
(test_gpu_shared_decode's bound, which covers scores, exponential and
additions too), or, below fp16's smallest step 2^-24, by half of that step.
The weights enter the products times 2^7 (relative to a row's running maximum,
which the largest score passes by 2^8 at most), so half a step is at most
2^-32 of the largest weight: 2^-32 / L a small token, with L the sum of a
row's weights relative to the largest, against small weights of 2^-25.97 / L:
2^-6 of the output."""
import math

import numpy as np
import pytest
import torch

import kvflux_b200 as kv
from test_gpu_shared_decode import FORMS, Batch

pytestmark = pytest.mark.gpu

HD = 64
KEY = 2.25  # score 64 * 2.25 / 8 = 18, 25.97 in base 2


def small_weights(groups, lens, room, group):
    b = Batch(groups, lens, 2, group, HD, dtype="float16", room=room)
    live = ~torch.isnan(b.k)
    b.k[live], b.v[live] = 0.0, 1.0
    first = live[:, :, 0, 0]
    b.k[:, :, 0][first] = KEY
    b.v[:, :, 0][first] = 0.0
    b.q.fill_(1.0)
    for d, h in ((b.dk, b.k), (b.dv, b.v), (b.dq, b.q)):
        d.copy_(h)
    return b


@pytest.mark.parametrize("group", [4, 9])
@pytest.mark.parametrize("groups,lens,room", FORMS + [([(40, 2064)], [2064 + 3 * i for i in range(40)], 0)])
def test_small_weights_count(cuda, groups, lens, room, group):
    kv.device_status(0, clear=True)
    b = small_weights(groups, lens, room, group)
    got = b.run().double()
    assert kv.device_status(0) == 0
    weight = math.exp(-HD * KEY / math.sqrt(HD))
    for r, n in enumerate(lens):
        large = -(-n // 16)
        want = (n - large) * weight / (large + (n - large) * weight)
        a = HD * KEY / math.sqrt(HD)
        tol = want * (2.0**-6 + 2 * a * (2.0**-23 + HD * 2.0**-23) + 2.0**-23 + 2.0**-21 + n * 2.0**-23)
        assert float((got[r] - want).abs().max()) <= tol, (r, n, float(got[r].min()), float(got[r].max()), want)


@pytest.mark.parametrize("step", [8.0, 16.0])
@pytest.mark.parametrize("pages", [4, 8])  # a warp's next page, a tile of the prefix
@pytest.mark.parametrize("groups,lens,room", FORMS)
def test_large_weights_stay_in_range(cuda, groups, lens, room, pages, step):
    """Tolerance: a sum of pairs (2^-23) against the sum of what they stand for, n additions each."""
    kv.device_status(0, clear=True)
    b = Batch(groups, lens, 2, 4, HD, dtype="float16", room=room)
    live = ~torch.isnan(b.k[:, :, :, 0])
    b.k[live], b.v[live] = 0.0, 1.0
    b.k[:, :, :, 0][live] = 2.0**11
    scale = math.sqrt(HD) * math.log(2)  # base-2 scores of q k
    b.q.fill_(0.0)
    b.q[:, :, 0], b.q[:, :, 1] = 2.0**15 * scale, step * scale
    for r in range(len(lens)):
        for j in range(-(-lens[r] // 16)):
            page = int(b.table[r, j])
            b.k[page, :, :, 1][live[page]] = float(j // pages)
    for d, h in ((b.dk, b.k), (b.dv, b.v), (b.dq, b.q)):
        d.copy_(h)
    got = b.run().double()
    assert kv.device_status(0) == 0
    for r, n in enumerate(lens):
        assert float((got[r] - 1).abs().max()) <= 2.0**-23 + 2 * n * 2.0**-23, r
