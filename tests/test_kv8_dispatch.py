"""The 8-bit KV cache's kernels at the sizes where a call takes another path: blocks of four tokens on
append, one list of key blocks shared by all warps and its join, keys of a prompt split over blocks.

References, checks and tolerances are those of test_kv8.py.
"""
import pytest
import torch

import test_kv8 as base
from vsa_lm_b200 import kernels as K


def spread(B, top, seed=0, idle=()):
    """B lengths in [0, top], `top` among them, -1 for the idle sequences."""
    lens = torch.randint(0, top + 1, (B,), generator=torch.Generator().manual_seed(seed)).tolist()
    lens[B // 2], lens[0] = top, 0
    for b in idle:
        lens[b] = -1
    return tuple(lens)


# From 148 * 8 tokens on a block takes four: the last block with one to four of them, rows of a thread that run
# over the ends of tokens (24, 25 and 3 rows a token)
APPEND = [
    (1184, 1, 16, 4, 64, 50, 60, True, True, None),
    (1185, 1, 15, 5, 128, 7, 9, False, True, None),
    (37, 32, 8, 8, 128, 100, 140, True, True, spread(37, 100, 1, (3, 36))),
    (9, 135, 1, 1, 64, 0, 140, True, True, None),
    (2, 593, 1, 1, 128, 3, 600, False, False, (7, -1)),
    (3, 397, 15, 5, 64, 20, 500, False, True, (103, 0, 11)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND)
def test_append_of_many_tokens(case):
    assert case[0] * case[1] >= 148 * 8
    base.test_append_matches_64_bits(case)


def check(B, T, H, HKV, HD, n, cap, lens, **kw):
    """A call over a cache that is poison past each sequence's rows; the workspace says whether it was split."""
    data, scale = base.random_cache(7, B, HKV, cap, HD)
    top = max(lens) if lens else n
    for b in range(B):
        s = n if lens is None else max(lens[b], -T)
        data[:, b, :, s + T:] = 127
        scale[:, b, :, s + T:] = float("nan")
    q = base.randn(8, B, T, H, HD, dtype=torch.bfloat16)
    L = torch.tensor(lens, dtype=torch.int32).cuda() if lens else None
    status = K.DeviceStatus("cuda")
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n, lens=L, status=status, **kw).cpu()
    assert int(status.word) == 0 and top + T <= cap
    base.check_attend(q, data, scale, n, lens, HD ** -0.5, y)


RUNS = [
    # B, T, H, HKV, HD, n, cap, lens
    (40, 1, 32, 8, 128, 700, 720, spread(40, 700, 1, (5, 6, 39))),    # 320 heads; runs that take whole short heads
    (160, 1, 8, 1, 64, 90, 91, spread(160, 90, 2, (1,) + tuple(range(64, 100)))),   # 32 idle in a row
    (20, 1, 16, 8, 128, 700, 701, None),                              # 160 heads, 13 partial sums of each or so
    (75, 1, 14, 2, 64, 64, 80, None),                                 # 3 blocks a head: one or two runs of each
    (1, 1, 8, 2, 128, 9000, 9001, None),                              # 2 heads, hundreds of partial sums of each
    (1, 4, 4, 1, 128, 4000, 4100, None),                              # 16 rows
    (3, 2, 16, 1, 64, 2000, 2100, (2000, -1, 33)),                    # 32 rows: two tiles of 16
    (50, 3, 16, 4, 64, 250, 300, spread(50, 250, 3, (0, 49))),        # 12 rows of 200 heads
    (40, 1, 8, 4, 128, 10, 400, spread(40, 399, 4)),                  # lengths above the expected one
    (160, 2, 5, 1, 128, 0, 2, None),                                  # nothing cached: heads of one block
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", RUNS)
def test_few_rows_in_runs(case):
    B, T, H, HKV, HD, n = case[:6]
    assert T * H // HKV <= 32 and K._attend_workspace(B, T, H, HKV, HD, n) > 0
    check(*case)


SPLIT = [
    (1, 64, 8, 2, 128, 3000, 3100, None),
    (2, 70, 8, 1, 64, 3000, 3072, (3000, 5)),        # most splits of the second sequence have no keys
    (2, 33, 4, 4, 128, 2900, 2933, (-1, 2900)),
    (1, 300, 4, 4, 64, 1024, 1400, None),            # 300 rows: two tiles of 128 and one of 44
    (3, 40, 2, 2, 128, 1500, 1600, (0, 1499, 700)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", SPLIT)
def test_prompt_keys_split_over_blocks(case):
    B, T, H, HKV, HD, n = case[:6]
    assert T * H // HKV > 32 and K._attend_workspace(B, T, H, HKV, HD, n) > 0
    check(*case)


@pytest.mark.gpu
def test_runs_of_idle_sequences_only():
    B, H, HKV, HD = 40, 16, 4, 64
    data, scale = base.new_cache(B, HKV, 32, HD)
    lens = torch.full((B,), -1, dtype=torch.int32).cuda()
    assert K._attend_workspace(B, 1, H, HKV, HD, 20) > 0
    y = K.kv8_attend(q=torch.ones(B, 1, H, HD, dtype=torch.bfloat16, device="cuda"), data=data, scale=scale, n=20, lens=lens)
    assert bool((y == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,HKV,HD,n", [(30, 1, 32, 8, 128, 300), (1, 40, 4, 2, 64, 2000)])
def test_device_position_in_runs_and_splits(B, T, H, HKV, HD, n):
    data, scale = base.random_cache(16, B, HKV, n + T + 40, HD)
    q = base.randn(15, B, T, H, HD, dtype=torch.bfloat16)
    pos = K.DevicePosition("cuda")
    pos.ref, pos.span = 100, 41
    pos.set(133)
    assert K._attend_workspace(B, T, H, HKV, HD, n) > 0
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n, dev_pos=pos).cpu()
    base.check_attend(q, data, scale, n + 33, None, HD ** -0.5, y)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    (3, 1, 8, 2, 128, 10, 400, (399, -1, 77)),       # a block per head
    (2, 60, 4, 2, 64, 10, 900, (840, 3)),            # prompt kernel
])
def test_lengths_above_the_expected_one(case):
    check(*case)
