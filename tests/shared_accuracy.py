"""How far attention over pairs of 16-bit operands is from 64 bits on normal
inputs, as a bound on the root mean square error, and a restatement of it on
the CPU (Q and the weights as hi + lo, or as hi alone) to try the bound on.

With o = sum p_t v_t, independent v and independent relative errors e_t of the
weights, rms(error) / rms(o) = rms(e_t). A bf16 pair is off by at most 2^-17
of itself (rms at most 2^-17 / sqrt 3 = 4.4e-6). In a score sum q_i k_i /
sqrt(hd) of standard normal values the errors of q add up to the same rms, as
a relative error of the weight; the weight's own pair adds another: 6.2e-6
together. Sums that truncate, of 16 products at a time: a score's 2 hd / 16,
each by at most 2^-23 of values of a few units, 2e-6 to 4e-6; those of O, at
most 128 a sum (8 tiles of 128 tokens, or a warp's pages of a split), by half
of 2^-23 on average, 7.6e-6. Together sqrt(6.2^2 + 4^2 + 7.6^2) = 10.6e-6,
below BOUND = 2^-16 = 15.3e-6. fp16 pairs (2^-23) are off by the sums alone.
A single operand is off by up to 2^-8 (bf16) or 2^-11 (fp16) of itself, rms
2.3e-3 and 2.8e-4 at a binade's lower end and about 0.7 of that over a binade:
above the bound by 10 and more."""
import torch

BOUND = 2.0**-16


def rms_error(got, want):
    return float(((got - want).square().mean() / want.square().mean()).sqrt())


def pair(x, dtype, lo=True):
    hi = x.to(dtype).double()
    return hi + (x - hi).to(dtype).double() if lo else hi


def attend(q, k, v, dtype, q_lo=True, p_lo=True):
    """Attention in 64 bits but for Q and the weights, which are 16-bit pairs or single values."""
    s = pair(q / q.shape[-1] ** 0.5, dtype, q_lo) @ k.transpose(-1, -2)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (pair(p, dtype, p_lo) @ v) / p.sum(-1, keepdim=True)
