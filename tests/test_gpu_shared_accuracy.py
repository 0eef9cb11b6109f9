"""Root mean square error of kvfx_decode_shared against 64 bits, with normal
inputs, where the worst-case bounds of test_gpu_shared_decode leave room for
operands of half the bits. The bound and its derivation: shared_accuracy.py."""
import pytest
import torch

import kvflux_b200 as kv
from shared_accuracy import BOUND, rms_error
from test_gpu_shared_decode import Batch

pytestmark = pytest.mark.gpu

CASES = [  # groups, lens, heads, q_group, hd, room
    ([(4, 64)], [64, 80, 100, 300], 2, 4, 128, 0),                                # one launch, row by row
    ([(8, 528)], [529 + i for i in range(8)], 2, 4, 64, 0),
    ([(8, 2064)], [2065 + 9 * i for i in range(8)], 2, 4, 64, 0),                 # prefix; tails that join it
    ([(8, 4096), (2, 2048)], [4097 + 5 * i for i in range(8)] + [2049, 2200], 2, 5, 128, 0),
    ([(40, 8192)], [8192 + i for i in range(40)], 1, 8, 128, 0),                  # three query tiles
    ([(3, 1040)], [9000, 1041, 5000], 2, 9, 64, 0),                               # several splits and the merge kernel
    ([(2, 32768)], [32769, 33000], 1, 4, 128, 0),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("groups,lens,heads,group,hd,room", CASES)
def test_errors_are_those_of_pairs(cuda, groups, lens, heads, group, hd, room, dtype):
    kv.device_status(0, clear=True)
    b = Batch(groups, lens, heads, group, hd, dtype=dtype, room=room)
    got = b.run()
    assert kv.device_status(0) == 0
    for r, n in enumerate(lens):
        t = torch.arange(n)
        page, off = torch.from_numpy(b.table[r].view("int64"))[t // 16], t % 16
        k, v = (x[page, :, off].double().permute(1, 0, 2) for x in (b.k, b.v))
        q = b.q[r].double().view(heads, -1, hd)
        want = torch.softmax(q @ k.transpose(1, 2) / hd**0.5, -1) @ v
        error = rms_error(got[r].double().view(want.shape), want)
        print(dtype, hd, n, error)
        assert error < BOUND, (r, n, error)
