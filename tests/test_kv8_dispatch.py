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
