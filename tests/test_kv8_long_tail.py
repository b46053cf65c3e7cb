"""One key holds nearly all of the probability, and very many keys far below it hold the rest: the rest is
what the output is made of in the dimensions where that key's value is zero.

Tolerance: weights are rounded to f16 at 2^-11 of themselves, and where they are below f16's normal range to within
2^-32 of the largest weighted value (a weight of 1 stands at 2^7 or more in f16, whose smallest step is 2^-24). The
scores are exact here but for their fp32 rounding (2^-22 in the weight at a score of 20).
"""
import math

import pytest
import torch

import test_kv8 as base
from vsa_lm_b200 import kernels as K


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,HKV,HD,n", [
    (1, 1, 4, 1, 64, 131071),         # split over the machine: the first key is in one of many partial sums
    (1, 40, 1, 1, 128, 131032),
    (230, 1, 16, 8, 64, 8191),        # a warp walks whole heads
    (250, 5, 8, 8, 128, 4091),
    (77, 40, 2, 2, 64, 65496),        # a block walks a whole head
    (160, 33, 1, 1, 128, 30000),
])
@pytest.mark.parametrize("bits", [25.4, 26.7, 22.0])
def test_tail_far_below_the_first_key(B, T, H, HKV, HD, n, bits):
    g = torch.Generator().manual_seed(31)
    data = torch.zeros(2, 1, 1, n + T, HD, dtype=torch.int8)
    data[0, 0, 0, 0, 0] = 127                                 # only this key has a component along the queries
    data[0, 0, 0, 1:, 1:] = torch.randint(-127, 128, (n + T - 1, HD - 1), generator=g, dtype=torch.int8)
    data[1, 0, 0, 0, 0] = 127
    data[1, 0, 0, 1:, 1:] = torch.randint(0, 51, (n + T - 1, HD - 1), generator=g, dtype=torch.int8)
    q = torch.zeros(B, T, H, HD, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    sm = bits * math.log(2.0) / 127                           # the other keys weigh 2^-bits of the first
    y = K.kv8_attend(q=q.cuda(), data=data.cuda().expand(2, B, HKV, n + T, HD).contiguous(),
                     scale=torch.ones(2, B, HKV, n + T, device="cuda"), n=n, sm_scale=sm).cpu().view(B, T, H, HD)
    v = data[1, 0, 0].double()
    below = v[1:].cumsum(0)                                   # of the tail, up to each key
    w = math.exp(-float(torch.tensor(sm, dtype=torch.float32)) * 127)
    for t in range(T):
        keys = n + t                                          # of the tail that token t sees
        ref = ((v[0] + w * below[keys - 1]) / (1 + w * keys)).expand(B, H, HD)
        assert base.rounded_within(y[:, t], ref, (2 ** -11 + 2 ** -18) * ref.abs() + keys * 2 ** -32 * 127), t
