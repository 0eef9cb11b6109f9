"""The bound that test_gpu_shared_accuracy holds the kernels to, on the CPU
restatement: pairs stay well inside it, and a dropped low half of Q or of the
weights does not pass."""
import pytest
import torch

from shared_accuracy import BOUND, attend, rms_error

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def case(n, hd, dtype, rows=16):
    gen = torch.Generator().manual_seed(n + hd)
    q = torch.randn(rows, hd, generator=gen).double()
    k, v = (torch.randn(n, hd, generator=gen).to(TYPES[dtype]).double() for _ in range(2))
    want = torch.softmax(q @ k.T / hd**0.5, -1) @ v
    return q, k, v, want


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,hd", [(100, 128), (529, 64), (2065, 64), (4097, 128), (32769, 128)])
def test_pairs_pass_and_single_operands_do_not(n, hd, dtype):
    q, k, v, want = case(n, hd, dtype)
    t = TYPES[dtype]
    assert rms_error(attend(q, k, v, t), want) < BOUND / 2
    assert rms_error(attend(q, k, v, t, q_lo=False), want) > 5 * BOUND
    assert rms_error(attend(q, k, v, t, p_lo=False), want) > 5 * BOUND
